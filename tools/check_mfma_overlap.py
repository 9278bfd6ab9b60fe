#!/usr/bin/env python3
"""Scan the gfx950 assembly of the HIP sources for MFMA instructions whose destination tuple PARTIALLY overlaps
their accumulator input (D != C but sharing registers).  ROCm 7.2 emits these for v_mfma_f32_16x16x32_bf16 builtins;
on MI355X they produced timing-dependent wrong results in the conv phase of the training kernel (DESIGN.md,
"compiler hazard").  The bf16x3 path therefore issues that instruction as tied inline asm; this script is the guard
that no builtin-generated instance is left, and that nothing touches the result of such an asm product before it is there.  Usage: tools/check_mfma_overlap.py [file.hip ...]   (exit 1 on a hit)"""
import os, re, subprocess, sys, tempfile
from concurrent.futures import ThreadPoolExecutor

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "purejaxql_amd", "csrc")
PAT = re.compile(r'(v_mfma_\w+)\s+([av])\[(\d+):(\d+)\],\s*[av]\[\d+:\d+\],\s*[av]\[\d+:\d+\],\s*([av])\[(\d+):(\d+)\]')


def scan(asm_path):
    hits, cur = [], "?"
    for ln, line in enumerate(open(asm_path), 1):
        if line.startswith("_Z") and ":" in line:
            cur = line.split(":")[0]
        m = PAT.search(line)
        if not m:
            continue
        dk, d0, d1, ck, c0, c1 = m.group(2), int(m.group(3)), int(m.group(4)), m.group(5), int(m.group(6)), int(m.group(7))
        if dk == ck and (d0, d1) != (c0, c1) and not (d1 < c0 or c1 < d0):
            hits.append((cur, ln, line.strip()))
    return hits


REG = re.compile(r'\bv(?:\[(\d+):(\d+)\]|(\d+)\b)')
WAIT = 11      # wait states between v_mfma_f32_16x16x32_bf16 (8 passes) and another instruction's access to its result
LABEL = re.compile(r'^([.\w$]+):')


def _regs(text):
    out = set()
    for lo, hi, one in REG.findall(text):
        out.update(range(int(lo), int(hi) + 1) if lo else (int(one),))
    return out


def _blocks(lines):
    """[(label, [(line number, mnemonic, operands)], successors)] of one kernel's text"""
    blocks, cur = [], ["", [], set()]
    for ln, line in lines:
        line = line.split(";")[0].strip()
        m = LABEL.match(line)
        if m:
            cur[2].add(m.group(1))
            blocks.append(cur)
            cur = [m.group(1), [], set()]
            continue
        if not line or line.startswith("."):
            continue
        op, _, rest = line.partition(" ")
        cur[1].append((ln, op, rest))
        if op.startswith("s_cbranch") or op == "s_branch":
            cur[2].add(rest.strip())
            if op == "s_branch":
                blocks.append(cur)
                cur = ["after line %d" % ln, [], set()]
        elif op == "s_endpgm":
            blocks.append(cur)
            cur = ["after line %d" % ln, [], set()]
    return blocks + [cur]


def _walk(block, left, hits):
    """Runs a block from the registers that still wait ({register: wait states}); what waits behind every branch and at its end"""
    out, left = {}, dict(left)

    def to(label):
        have = out.setdefault(label, {})
        for r, n in left.items():
            have[r] = max(have.get(r, 0), n)

    for ln, op, rest in block[1]:
        if op == "v_mfma_f32_16x16x32_bf16":
            d, a, b, c = (_regs(x) for x in re.split(r",\s*(?![^\[]*\])", rest)[:4])
            if (a | b) & set(left) or (c != d and (c | d) & set(left)):
                hits.append((ln, op + " " + rest))
        elif _regs(rest) & set(left):
            hits.append((ln, op + " " + rest))
        passed = int(rest) + 1 if op == "s_nop" else 1
        left = {r: n - passed for r, n in left.items() if n > passed}
        if op == "v_mfma_f32_16x16x32_bf16":
            left.update({r: WAIT for r in d})
        if op.startswith("s_cbranch") or op == "s_branch":
            to(rest.strip())
    for label in block[2]:
        if not any(op.startswith(("s_cbranch", "s_branch")) and rest.strip() == label for _, op, rest in block[1]):
            to(label)
    return out


def scan_unfinished(asm_path):
    """The bf16 products are asm, whose results the compiler takes for ready at once: every access to one but the next product of its
    chain has to lie WAIT wait states behind it, on every path (a copy or a spill that the compiler puts between is found here)."""
    hits, kernel, cur = [], None, []
    kernels = []
    for ln, line in enumerate(open(asm_path), 1):
        if line.startswith("_Z") and ":" in line:
            kernel, cur = line.split(":")[0], []
            kernels.append((kernel, cur))
        elif line.startswith(".Lfunc_end"):
            kernel = None
        elif kernel:
            cur.append((ln, line))
    for name, lines in kernels:
        blocks = _blocks(lines)
        at = {b[0]: {} for b in blocks}
        todo, found = [b for b in blocks], set()
        by = {b[0]: b for b in blocks}
        while todo:
            b = todo.pop()
            mine = []
            for label, left in _walk(b, at[b[0]], mine).items():
                if label not in at:
                    continue
                more = {r: n for r, n in left.items() if n > at[label].get(r, 0)}
                if more:
                    at[label].update(more)
                    todo.append(by[label])
            found.update(mine)
        hits += [(name, ln, text) for ln, text in sorted(found)]
    return hits


M0_OK = re.compile(r'^\s*s_mov_b32 m0, s\d+\s*$')


def scan_m0(asm_path):
    """pqn_qnet_pos.hip leaves M0 holding the LDS-DMA destination (pos_dma16 does not save / restore it since round 6): every
    mention of m0 in its assembly must be one of those writes -- nothing may READ it (s_movrel, sendmsg, GWS, v_readlane m0 ...)."""
    return [(ln, line.strip()) for ln, line in enumerate(open(asm_path), 1)
            if re.search(r'\bm0\b', line.split(";")[0]) and not M0_OK.match(line.split(";")[0])]


def assembly(f, out):
    """The gfx950 assembly of a HIP source, as the Makefile builds it"""
    extra = ["-fno-slp-vectorize"] if os.path.basename(f) == "pqn_qnet_pos.hip" else []
    subprocess.run(["/opt/rocm/bin/hipcc", "-O3", "-std=c++17", "-fPIC", "--offload-arch=gfx950", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", *extra, "--cuda-device-only", "-S", f, "-o", out], check=True, cwd=CSRC, stderr=subprocess.DEVNULL)


def scanned(f):
    """(partial overlaps, early accesses, uses of M0) of a source"""
    with tempfile.TemporaryDirectory() as td:
        out = os.path.join(td, "x.s")
        assembly(f, out)
        return scan(out), scan_unfinished(out), scan_m0(out) if os.path.basename(f) == "pqn_qnet_pos.hip" else []


def main():
    files = [os.path.abspath(f) for f in sys.argv[1:]] or [os.path.join(CSRC, f) for f in sorted(os.listdir(CSRC)) if f.endswith(".hip")]
    bad = 0
    with ThreadPoolExecutor(4) as pool:
        for f, (hits, early, m0) in zip(files, pool.map(scanned, files)):
            name = os.path.basename(f)
            if name == "pqn_qnet_pos.hip":
                print("%-20s %d uses of M0 other than the LDS-DMA destination writes" % (name, len(m0)))
                for ln, l in m0[:8]:
                    print("    line %d  %s" % (ln, l))
            print("%-20s %d partially overlapping MFMA D/C" % (name, len(hits)))
            print("%-20s %d accesses to the result of a bf16 product within %d wait states" % (name, len(early), WAIT))
            for k, ln, l in hits[:12] + early[:12]:
                print("    %s:%d  %s" % (k[:50], ln, l))
            bad += len(hits) + len(early) + len(m0)
    sys.exit(1 if bad else 0)


if __name__ == "__main__":
    main()
