"""Matrix results read too early, found in a listing of gfx950 code.

A v_mfma instruction's result is in its registers only some wait states later (an instruction is one, s_nop n is n + 1),
and nothing in the hardware holds an earlier reader back: the compiler has to keep the distance.  early_reads() follows
every path through a listing, branches included, with the states that each register still needs (where paths meet, the
most that any of them needs), and returns what reads or overwrites one before.

A product that takes a result as its addend is not looked at (sums over products are chains of those, which need
none or two states); one that takes it as a factor is.
"""
import re

# wait states from the product to the first reader: of 4 passes, of 8, and of 8 in f32 (the least that the compiler
# leaves between the two in straight code)
STATES = {"f32_16x16x16_f16": 8, "f32_16x16x32_f16": 8, "i32_16x16x32_i8": 8, "i32_16x16x64_i8": 8,
          "f32_32x32x16_f16": 12, "f32_16x16x4_f32": 10}

_WIDE = re.compile(r"\b([va])\[(\d+):(\d+)\]")
_ONE = re.compile(r"(?<![\w\[:.])([va])(\d+)\b")
_OPERAND = re.compile(r"[va]\[\d+:\d+\]|[^,\s]+")


def _regs(text):
    out = {(f, n) for f, a, b in _WIDE.findall(text) for n in range(int(a), int(b) + 1)}
    out.update((f, int(n)) for f, n in _ONE.findall(text))
    return out


def functions(listing):
    """(name, [instruction or 'label:']) of every function of the listing (llvm-objdump --symbolize-operands)."""
    name, code = None, []
    for line in listing.splitlines():
        m = re.match(r"(?:[0-9a-f]+ )?<(\w+)>:", line)
        if m and re.fullmatch(r"L\d+", m.group(1)):
            code.append(m.group(1) + ":")
        elif m:
            if name is not None:
                yield name, code
            name, code = m.group(1), []
        elif name is not None:
            text = line.split("//")[0].strip()
            if text and not text.startswith(("Disassembly", ".")):
                code.append(text)
    if name is not None:
        yield name, code


def early_reads(code):
    """[(index, instruction, wait states short)] of a function."""
    labels = {t[:-1]: i for i, t in enumerate(code) if t.endswith(":")}
    at, found = [None] * len(code), {}
    work = [(0, {})]  # places to go on from, and the states that registers still need there
    while work:
        i, need = work.pop()
        while i < len(code):
            text = code[i]
            if text.endswith(":"):
                i += 1
                continue
            if at[i] is not None:
                need = {r: max(need.get(r, 0), at[i].get(r, 0)) for r in need.keys() | at[i].keys()}
                if need == at[i]:
                    break
            at[i] = need
            op, _, rest = text.partition(" ")
            reads, result = rest, None
            if op.startswith(("v_mfma", "v_smfma")):
                result, a, b = _OPERAND.findall(rest)[:3]
                reads, shape = a + " " + b, op.split("_", 2)[2]
                if shape not in STATES:
                    raise ValueError(f"{op}: the wait states of its result are not known")
            short = max((need.get(r, 0) for r in _regs(reads)), default=0)
            if short > 0:
                found[i] = max(short, found.get(i, 0))
            step = int(rest.split()[0], 0) + 1 if op == "s_nop" else 1
            need = {r: v - step for r, v in need.items() if v > step}
            if result is not None:
                need.update((r, STATES[shape]) for r in _regs(result))
            if op in ("s_endpgm", "s_setpc_b64"):
                break
            if op == "s_branch":
                i = labels[rest.split()[0]]
                continue
            if op.startswith("s_cbranch"):
                work.append((labels[rest.split()[0]], need))
            i += 1
    return [(i, code[i], short) for i, short in sorted(found.items())]
