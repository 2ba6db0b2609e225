#!/usr/bin/env python3
"""Audits the device assembly of a HIP source for reads of a matrix instruction's result that come too
early.  On gfx950 the result of a v_mfma is not interlocked against vector instructions: a read needs (passes + 3)
wait states after the instruction (passes + 2 for fp32 inputs), which the compiler fills with s_nop.  hipcc 7.2 has been
seen to leave them out in front of v_accvgpr_read where the matrix instruction ends a loop and its accumulator sits in
AGPRs: the first element of each accumulator then holds the value before the last product.

  audit_mfma_waits.py FILE.s [...]      lists the findings, exit code 1 if there are any"""
import re
import sys

REG = re.compile(r"\b([av])(?:\[(\d+):(\d+)\]|(\d+))(?![\w\[])")
LABEL = re.compile(r"^(\.?\w[\w.$]*):")


def regs(text):
    out = set()
    for m in REG.finditer(text):
        lo = int(m.group(2) or m.group(4))
        hi = int(m.group(3) or m.group(4))
        out.update((m.group(1), i) for i in range(lo, hi + 1))
    return out


def wait_states(op):
    """Needed between this matrix instruction and a vector read of its result."""
    m = re.match(r"v_mfma_\w*?f32_(\d+)x(\d+)x(\d+)_?(\w+)", op)
    a, k, kind = int(m.group(1)), int(m.group(3)), m.group(4)
    if kind.startswith("f32"):
        passes = {4: 2, 16: 8, 32: 16}[a]
        return passes + 2
    passes = {16: 4, 32: 8}[a] * (1 if (a, k) in ((16, 16), (16, 32), (32, 8), (32, 16)) else 2)
    return passes + 3


def functions(lines):
    start = None
    for n, line in enumerate(lines):
        m = re.match(r"^(_Z\w+|\w+):\s*(;.*)?$", line)
        if m and not line.startswith(".L"):
            start = (m.group(1), n)
        if line.startswith(".Lfunc_end") and start:
            yield start[0], start[1], n
            start = None


def audit(lines, a, b):
    ins, labels = [], {}
    for n in range(a, b):
        text = lines[n].split(";")[0].strip()
        m = LABEL.match(lines[n])
        if m:
            labels[m.group(1)] = len(ins)
            continue
        if text and not text.startswith("."):
            ins.append((n, text))
    found = []
    for p, (n, text) in enumerate(ins):
        if not text.startswith("v_mfma"):
            continue
        op, rest = text.split(None, 1)
        dst = regs(rest.split(",")[0])
        need = wait_states(op)
        seen, todo = {}, [(p + 1, 0, dst)]
        while todo:
            q, done, live = todo.pop()
            while q < len(ins) and done < need and live:
                if seen.get(q, 1 << 30) <= done:
                    break
                seen[q] = done
                t = ins[q][1]
                o = t.split(None, 1)[0]
                args = t.split(None, 1)[1].split(",") if " " in t or "\t" in t else []
                if o == "s_nop":
                    done += int(args[0]) + 1
                    q += 1
                    continue
                if o == "s_endpgm":
                    break
                if o.startswith("s_branch") or o.startswith("s_cbranch"):
                    to = labels.get(args[0].strip())
                    if to is not None:
                        todo.append((to, done + 1, live))
                    if o == "s_branch":
                        break
                elif o.startswith("v_mfma"):
                    read = regs(",".join(args[1:3]))  # A and B; the accumulator operand is forwarded
                    if read & live:
                        found.append((lines[n].strip(), ins[q][1], need - done))
                        break
                    live = live - regs(args[0])
                elif args:
                    writes = o.startswith(("v_", "global_load", "ds_read", "buffer_load"))
                    read = regs(",".join(args[1:] if writes else args))
                    if read & live:
                        found.append((lines[n].strip(), ins[q][1], need - done))
                        break
                    if writes and o.startswith("v_"):
                        live = live - regs(args[0])
                done += 1
                q += 1
    return found


def audit_file(path):
    lines = open(path).read().split("\n")
    return {name: f for name, a, b in functions(lines) if (f := audit(lines, a, b))}


if __name__ == "__main__":
    bad = 0
    for path in sys.argv[1:]:
        for name, f in audit_file(path).items():
            for mfma, reader, missing in f:
                print(f"{path}: {name}: {missing} wait states short: {mfma}  ->  {reader}")
                bad += 1
    sys.exit(1 if bad else 0)
