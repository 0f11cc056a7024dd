"""Check of the compiler's assembly output for this library's kernels (`make check`).

Direct loads to LDS (dma.h) are inline assembly, and the compiler keeps no distance in front of what
it does not know to be a load.  A load that takes its base from a scalar register may follow a vector
instruction that wrote this register (readfirstlane, readlane, a comparison) only behind five
wait states; short of them it reads what the register held before, and goes to a wild address.  A
base that scalar instructions computed needs none.  This script finds direct loads that come too soon,
along straight-line code and from the end of a block into the one that follows it.

usage: check_sgpr_reads.py file.s [file.s ...]    (exit status 1 if anything is found)
"""
import re
import sys

NEED = 5
READS_ONLY = ("s_cmp", "s_bitcmp", "s_setpc", "s_setreg", "s_setvskip", "s_set_gpr_idx", "s_branch", "s_cbranch")  # their first operand is no destination


def sgprs(text):
    out = set()
    text = re.sub(r"\bvcc\b", "vcc_lo vcc_hi", text)
    out.update(name for name in ("vcc_lo", "vcc_hi") if name in text)
    for m in re.finditer(r"\bs\[(\d+):(\d+)\]", text):
        out.update(range(int(m.group(1)), int(m.group(2)) + 1))
    for m in re.finditer(r"\bs(\d+)\b", text):
        out.add(int(m.group(1)))
    return out


def scan(path):
    found, func, states, written = 0, "?", 0, {}
    for number, line in enumerate(open(path), 1):
        line = line.split(";")[0].rstrip()
        if line.endswith(":") and line.startswith("_Z"):
            func, written = line[:-1], {}
            continue
        text = line.strip()
        if not text or text.endswith(":") or text.startswith("."):
            continue
        op, _, rest = text.partition(" ")
        op, rest = op.split("\t")[0], rest or text.partition("\t")[2]
        if op == "s_nop":
            states += int(rest) + 1
            continue
        if op.startswith("global_load_lds"):
            soon = [states - written[r] for r in sgprs(rest) if r in written and states - written[r] < NEED]
            if soon:
                print(f"{path}:{number}: {func[:70]}\n    {text}\n    {min(soon)} wait states behind the write of its base")
                found += 1
        first = rest.split(",")[0]
        if op.startswith("v_"):
            for r in sgprs(first):
                written[r] = states + 1
        elif op.startswith("s_") and not op.startswith(READS_ONLY):
            for r in sgprs(first):
                written.pop(r, None)
        states += 1
    return found


if __name__ == "__main__":
    total = sum(scan(p) for p in sys.argv[1:])
    print(f"{total} direct loads too soon behind the write of their base")
    sys.exit(1 if total else 0)
