"""Builds the gfx950 operator library (``libdhellam_hip.so``) with hipcc.

The library is plain HIP behind a C ABI (``include/dhellam_hip.h``): no torch
headers, so a cross-compile needs only ROCm.  Objects go to ``build/`` and the
shared object to ``dhellam_amd/lib/`` (in-tree, so it is found next to the
package without installation).

Run as ``python -m dhellam_amd.build``.
"""
from __future__ import annotations

import os
import subprocess
import sys
import sysconfig
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG = Path(__file__).resolve().parent
ROOT = PKG.parent
CSRC = PKG / "csrc"
LIB_DIR = PKG / "lib"
LIB_PATH = LIB_DIR / "libdhellam_hip.so"
OBJ_DIR = ROOT / "build" / "obj"
GEN_DIR = ROOT / "build" / "gen"          # sources that are written by programs: attn_loops.inc

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"

# -packed-fp32-ops is switched off: the compiler would otherwise form packed
# fp32 VALU instructions from scalar float code.
CXXFLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-fno-gpu-rdc",
    "-Wall",
    "-Wno-unused-function",
    "-Wno-unknown-pragmas",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{ROOT / 'include'}",
    f"-I{GEN_DIR}",
]


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.hip"))


def generate_sources() -> None:
    """Writes ``attn_loops.inc``: the main loops of the attention kernels with one wavefront on a SIMD (``csrc/attn_loops.py``)."""
    GEN_DIR.mkdir(parents=True, exist_ok=True)
    subprocess.run([sys.executable, str(CSRC / "attn_loops.py"), str(GEN_DIR / "attn_loops.inc")], check=True)


def _compile(src: Path, verbose: bool) -> Path:
    obj = OBJ_DIR / (src.stem + ".o")
    cmd = [HIPCC, *CXXFLAGS, "-c", str(src), "-o", str(obj)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    # hipcc's host pass warns that it does not know the packed-fp32 feature; drop that line.
    err = "\n".join(l for l in res.stderr.splitlines() if "packed-fp32-ops" not in l)
    if res.returncode != 0:
        raise RuntimeError(f"hipcc failed for {src.name}:\n{err}")
    if err.strip() and verbose:
        print(err, file=sys.stderr)
    return obj


def build(verbose: bool = False, jobs: int | None = None) -> Path:
    """Compile every ``csrc/*.hip`` for gfx950 and link the shared library."""
    OBJ_DIR.mkdir(parents=True, exist_ok=True)
    LIB_DIR.mkdir(parents=True, exist_ok=True)
    generate_sources()
    srcs = sources()
    if not srcs:
        raise RuntimeError(f"no HIP sources under {CSRC}")
    jobs = jobs or min(8, len(srcs), os.cpu_count() or 1)
    with ThreadPoolExecutor(max_workers=jobs) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-fno-gpu-rdc",
           *map(str, objs), "-lhipblaslt", "-o", str(tmp)]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"link failed:\n{res.stderr}")
    os.replace(tmp, LIB_PATH)
    return LIB_PATH


def grouped_gemm_assembly() -> list:
    """The instantiations of ``grouped_gemm_w8_kernel`` as device assembly of ``grouped_gemm.hip``, a list of lines each."""
    import re
    import tempfile
    with tempfile.TemporaryDirectory() as td:
        out = Path(td) / "gg.s"
        cmd = [HIPCC, *[f for f in CXXFLAGS if f != "-fPIC"], "--cuda-device-only", "-S", str(CSRC / "grouped_gemm.hip"), "-o", str(out)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("hipcc -S failed for grouped_gemm.hip:\n" + res.stderr)
        lines = out.read_text().split("\n")
    starts = [i for i, l in enumerate(lines) if re.match(r"^_ZN2dh22grouped_gemm_w8_kernel\w+:", l)]
    if not starts:
        raise RuntimeError("no grouped_gemm_w8_kernel instantiation found in the assembly")
    # (a kernel may hold several s_endpgm)
    return [lines[a:next(i for i in range(a, len(lines)) if lines[i].startswith(".Lfunc_end"))] for a in starts]


def check_grouped_gemm_loops(verbose: bool = False) -> int:
    """The chip-filling grouped GEMM kernel (``grouped_gemm_w8_kernel``) copies its operands to LDS from assembly, which
    the compiler does not count: that no copy overtakes a fragment read and no read a copy rests on the order of reads,
    waits, copies and barriers that the source lays down.  This holds the generated code of every instantiation to it
    (``check_grouped_gemm_order``).  Returns the number of instantiations checked; raises on a violation."""
    kernels = grouped_gemm_assembly()
    for fn in kernels:
        body = check_grouped_gemm_order(fn)
        if verbose:
            print(f"checked {fn[0].split(':')[0]}: {body} lines", flush=True)
    return len(kernels)


def check_grouped_gemm_order(fn: list) -> int:
    """One instantiation of ``grouped_gemm_w8_kernel`` as assembly: the copies of the first two slices, published by the
    counted wait and a barrier before anything is read, and one more barrier for half of the wavefronts; the main loop (the
    innermost loop with 128 MFMAs: two slices) and, behind it, the last slice of an odd number.  In the slices, cut at their
    barriers, clusters of 16 MFMAs have to alternate with clusters of none, copies may stand in the latter only, each of these
    has to begin by waiting for the wavefront's earlier LDS reads, and where copies are published the wait for them is the one
    the source counts.  Behind the last slice everything has landed, past a barrier, before LDS is used again.  No scratch
    accesses, no copies of accumulators, and no register moves among MFMAs.  Returns the lines of the loop."""
    import re
    name = fn[0].split(":")[0]
    code = [l.split(";")[0].strip() for l in fn]
    labels = {m.group(1): i for i, l in enumerate(code) if (m := re.match(r"^(\.LBB\d+_\d+):", l))}
    mfmas = lambda part: sum("v_mfma" in x for x in part)
    barriers = lambda part: [i for i, x in enumerate(part) if x.startswith("s_barrier")]
    copies = lambda part: [i for i, x in enumerate(part) if x.startswith("buffer_load")]

    def need(ok, what):
        if not ok:
            raise RuntimeError(f"{name}: {what}")

    loops = []
    for i, l in enumerate(code):
        m = re.match(r"s_c?branch\w* (\.LBB\d+_\d+)", l)
        if m and m.group(1) in labels and labels[m.group(1)] < i and mfmas(code[labels[m.group(1)] + 1:i]) == 128:
            loops.append((labels[m.group(1)] + 1, i))
    need(loops, "no main loop with 128 MFMAs found (the kernel's structure changed: update check_grouped_gemm_order)")
    lo, hi = min(loops, key=lambda x: x[1] - x[0])
    plain = lambda part: [x for x in part if x and not x.endswith(":")]
    first, body, rest = plain(code[:lo]), plain(code[lo:hi]), plain(code[hi:])
    need(mfmas(first) == 0 and mfmas(rest) == 64, f"{mfmas(first)} and {mfmas(rest)} MFMAs before and behind the main loop, expected 0 and 64")

    def check_slices(clusters, where):
        total = 0
        for n, cl in enumerate(clusters):
            dma = copies(cl)
            need(mfmas(cl) == (16 if n % 2 else 0), f"{where}: cluster {n} holds {mfmas(cl)} MFMAs")
            need(not any("scratch_" in x or "v_accvgpr" in x for x in cl), f"{where}: scratch or accumulator copies in cluster {n}")
            total += len(dma)
            if n % 2:
                need(not dma, f"{where}: a copy among the MFMAs of cluster {n}")
                need(not any(x.startswith("v_mov_b") for x in cl), f"{where}: a register move among the MFMAs of cluster {n}")
                continue
            waits = [i for i, x in enumerate(cl) if x == "s_waitcnt lgkmcnt(0)"]
            reads = [i for i, x in enumerate(cl) if x.startswith("ds_read")]
            need(waits and not (reads and reads[0] < waits[0]) and not (dma and dma[0] < waits[0]),
                 f"{where}: cluster {n} does not begin with the wait for the earlier reads")
            need(all(cl[i].endswith("lds") for i in dma), f"{where}: a load to registers in cluster {n}")
            need(not dma or "s_waitcnt vmcnt(8)" in cl[dma[-1]:], f"{where}: cluster {n} publishes copies without the counted wait")
        need(total == len(clusters), f"{where}: {total} copies, expected {len(clusters)}")

    def cut(part):
        at = [-1] + barriers(part)
        return [part[x + 1:y] for x, y in zip(at, at[1:])], part[at[-1] + 1:]

    # the first two slices
    dma = copies(first)
    need(len(dma) == 16 and all(first[i].endswith("lds") for i in dma), f"{len(dma)} loads before the main loop, expected 16 copies")
    need("s_waitcnt vmcnt(0)" in first[:dma[0]], "the stores before the first copies are not waited for")
    behind = first[dma[-1] + 1:]
    bars = barriers(behind)
    need(len(bars) == 2, f"{len(bars)} barriers between the first copies and the main loop, expected 2")
    need("s_waitcnt vmcnt(8)" in behind[:bars[0]], "the first slice is published without the counted wait")
    reads = [i for i, x in enumerate(first) if x.startswith("ds_read")]
    need(reads and reads[0] > dma[-1] + 1 + bars[1], "a fragment is read before the first slice is published")
    # the loop
    clusters, head = cut(body)
    need(len(clusters) == 16, f"{len(clusters)} barriers in the main loop, expected 16")
    clusters[0] = head + clusters[0]                     # what follows the last barrier runs into the loop's head
    check_slices(clusters, "main loop")
    # the last slice of an odd number
    at = barriers(rest)
    need(len(at) >= 10, f"{len(at)} barriers behind the main loop, expected 10 and more")
    clusters, _ = cut(rest[:at[7] + 1])
    waits = [i for i, x in enumerate(clusters[0]) if x == "s_waitcnt lgkmcnt(0)"]    # (the blocks that the branches over it lead to)
    need(waits and not any(x.startswith("ds_read") for x in clusters[0][:waits[-1]]), "last slice: a read before the wait for the earlier ones")
    clusters[0] = clusters[0][waits[-1]:]
    check_slices(clusters, "last slice")
    # and what follows: the other half's barrier, the last copies, a barrier, and only then LDS again
    behind = rest[at[7] + 1:]
    used = next((i for i, x in enumerate(behind) if x.startswith(("ds_", "global_store", "buffer_load"))), len(behind))
    landed = next((i for i, x in enumerate(behind) if re.match(r"s_waitcnt vmcnt\(0\)", x)), len(behind))
    need(landed < used and any(landed < i < used for i in barriers(behind)), "LDS is used again before the last copies have landed")
    return len(body)


def mx_gemm_assembly() -> dict:
    """The instantiations of ``mx_w8_kernel`` and ``mx_t128_kernel`` as device assembly of ``mx_gemm.hip``, a list of lines each, by their
    mangled names."""
    import re
    import tempfile
    with tempfile.TemporaryDirectory() as td:
        out = Path(td) / "mx.s"
        cmd = [HIPCC, *[f for f in CXXFLAGS if f != "-fPIC"], "--cuda-device-only", "-S", str(CSRC / "mx_gemm.hip"), "-o", str(out)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("hipcc -S failed for mx_gemm.hip:\n" + res.stderr)
        lines = out.read_text().split("\n")
    starts = [i for i, l in enumerate(lines) if re.match(r"^_ZN2dh(12mx_w8|14mx_t128)_kernel\w+:", l)]
    return {lines[a].split(":")[0]: lines[a:next(i for i in range(a, len(lines)) if lines[i].startswith(".Lfunc_end"))] for a in starts}


def check_mx_gemm_loops(verbose: bool = False) -> int:
    """The tiled products of microscaled operands copy to LDS from assembly too, and form their sums in assembly: the generated code of every
    instantiation is held to the order that the source lays down (``check_mx_gemm_order``) and to the distances that the compiler does not keep
    for instructions it does not know (``check_mx_gemm_distances``).  Returns their number; raises on a violation."""
    kernels = mx_gemm_assembly()
    for name, fn in kernels.items():
        body = check_mx_gemm_order(name, fn)
        check_mx_gemm_distances(name, fn)
        if verbose:
            print(f"checked {name}: {body} lines", flush=True)
    return len(kernels)


def _mx_gemm_parts(name: str, fn: list):
    """The code of an instantiation before, in and behind its main loop (the innermost loop with the matrix instructions of two slices), and what a
    slice has: its matrix instructions, a wavefront's copies."""
    import re
    fa, fb = (int(x) for x in re.search(r"kernelILi(\d)ELi(\d)E", name).groups())
    two = fa == 4 and fb == 4
    rows = lambda bits: 2 if two or bits == 8 else 1                  # 1 KB copies of 64 rows
    copies = (2 if two else 1) + 2 * rows(fa) + 2 * rows(fb)
    slice_mfmas = 32 if "mx_w8" in name else 64 if "Lb1E" in name else 16
    code = [x for x in (l.split(";")[0].strip() for l in fn) if x]
    labels = {m.group(1): i for i, l in enumerate(code) if (m := re.match(r"^(\.LBB\d+_\d+):", l))}
    loops = []
    for i, l in enumerate(code):
        m = re.match(r"s_c?branch\w* (\.LBB\d+_\d+)", l)
        if m and m.group(1) in labels and labels[m.group(1)] < i and sum("v_mfma" in x for x in code[labels[m.group(1)] + 1:i]) == 2 * slice_mfmas:
            loops.append((labels[m.group(1)] + 1, i))
    if not loops:
        raise RuntimeError(f"{name}: no main loop with {2 * slice_mfmas} matrix instructions")
    lo, hi = min(loops, key=lambda x: x[1] - x[0])
    plain = lambda part: [x for x in part if not x.endswith(":")]
    return plain(code[:lo]), plain(code[lo:hi]), plain(code[hi:]), slice_mfmas, copies


def check_mx_gemm_order(name: str, fn: list) -> int:
    """One instantiation of ``mx_w8_kernel`` or ``mx_t128_kernel``: the first copies, published before anything is read; two slices in the main loop;
    and behind it the last slice of an odd number, held to the same.  Every copy goes to LDS.
    ``mx_w8_kernel``: 8 clusters a slice between barriers, every second one of 8 matrix instructions and no copy, the others beginning with the
    wait for the wavefront's earlier reads and ending, where they publish copies, with the counted wait.  ``mx_t128_kernel``: a slice begins with
    the waits for reads and copies and a barrier, and its copies go out behind that.  No scratch accesses in the loop, and behind the last slice the
    last copies are waited for before LDS is used again or the kernel ends.  Returns the lines of the loop."""
    first, body, rest, slice_mfmas, copies = _mx_gemm_parts(name, fn)
    eight = "mx_w8" in name
    mfmas = lambda part: sum("v_mfma" in x for x in part)
    copies_of = lambda part: [i for i, x in enumerate(part) if x.startswith("buffer_load")]
    reads_of = lambda part: [i for i, x in enumerate(part) if x.startswith("ds_read")]
    barriers = lambda part: [i for i, x in enumerate(part) if x.startswith("s_barrier")]

    def need(ok, what):
        if not ok:
            raise RuntimeError(f"{name}: {what}")

    def published(part, at):                       # the waits right before a barrier of mx_t128_kernel
        return part[at - 2:at] == ["s_waitcnt lgkmcnt(0)", "s_waitcnt vmcnt(0)"]

    def check_clusters(clusters, where):
        dma = 0
        for n, cl in enumerate(clusters):
            need(mfmas(cl) == (8 if n % 2 else 0), f"{where}: cluster {n} holds {mfmas(cl)} matrix instructions")
            need(not any("scratch_" in x for x in cl), f"{where}: scratch accesses in cluster {n}")
            at, waits, reads = copies_of(cl), [i for i, x in enumerate(cl) if x == "s_waitcnt lgkmcnt(0)"], reads_of(cl)
            dma += len(at)
            if n % 2:
                need(not at, f"{where}: a copy in cluster {n}, among matrix instructions")
                continue
            need(waits and not (reads and reads[0] < waits[0]) and not (at and at[0] < waits[0]),
                 f"{where}: cluster {n} does not begin with the wait for the earlier reads")
            need(not at or f"s_waitcnt vmcnt({copies})" in cl[at[-1]:], f"{where}: cluster {n} publishes copies without the counted wait")
        need(dma == len(clusters) // 8 * copies, f"{where}: {dma} copies in {len(clusters) // 8} slices of {copies}")

    need(all(x.endswith("lds") for part in (first, body, rest) for x in part if x.startswith("buffer_load")), "a buffer load to registers")
    need(mfmas(first) == 0 and mfmas(rest) == slice_mfmas, f"{mfmas(first)} and {mfmas(rest)} matrix instructions before and behind the main loop")
    # the first two slices' copies
    dma, reads, at = copies_of(first), reads_of(first), barriers(first)
    need(len(dma) == 2 * copies, f"{len(dma)} copies before the main loop, expected {2 * copies}")
    need(at and reads and reads[0] > at[0], "a fragment is read before the first slice is published")
    if eight:
        need(len(at) == 2 and at[0] > dma[-1] and f"s_waitcnt vmcnt({copies})" in first[dma[-1]:at[0]] and reads[0] > at[1],
             "the first slice is not published by the counted wait and a barrier, one more of half of the wavefronts behind it")
    else:
        need(len(at) == 1 and dma[copies - 1] < at[0] < dma[copies] and "s_waitcnt vmcnt(0)" in first[dma[copies - 1]:at[0]],
             "the first slice is not published by the wait for its copies and a barrier")
    # the main loop
    need(not any("scratch_" in x for x in body), "scratch accesses in the main loop")
    need(len(copies_of(body)) == 2 * copies, f"{len(copies_of(body))} copies in the main loop, expected {2 * copies}")
    at = barriers(body)
    if eight:
        need(len(at) == 16, f"{len(at)} barriers in the main loop, expected 16")
        clusters = [body[a + 1:b] for a, b in zip([-1] + at, at)]
        clusters[0] = body[at[-1] + 1:] + clusters[0]
        check_clusters(clusters, "main loop")
    else:
        need(len(at) == 2, f"{len(at)} barriers in the main loop, expected 2")
        need(all(published(body, b) for b in at), "a slice begins without the waits for reads and copies")
        for part in (body[at[0] + 1:at[1]], body[at[1] + 1:] + body[:at[0]]):
            need(mfmas(part) == slice_mfmas and len(copies_of(part)) == copies, "a slice's copies or matrix instructions are in another's place")
    # the last slice of an odd number
    at = barriers(rest)
    if eight:
        need(len(at) >= 9, f"{len(at)} barriers behind the main loop, expected 9 and more")
        clusters = [rest[a + 1:b] for a, b in zip([-1] + at, at[:8])]
        waits = [i for i, x in enumerate(clusters[0]) if x == "s_waitcnt lgkmcnt(0)"]      # (the blocks that the branches over it lead to)
        need(waits and not reads_of(clusters[0][:waits[-1]]), "last slice: a read before the wait for the earlier ones")
        clusters[0] = clusters[0][waits[-1]:]
        check_clusters(clusters, "last slice")
    else:
        need(len(at) >= 2 and published(rest, at[0]), "the last slice begins without the waits for reads and copies")
        part = rest[at[0] + 1:at[1]]
        need(mfmas(part) == slice_mfmas and len(copies_of(part)) == copies and not reads_of(rest[:at[0]]) and not any("scratch_" in x for x in part),
             "the last slice's reads, copies or matrix instructions are in another's place")
    last = max(i for i, x in enumerate(rest) if "v_mfma" in x)
    landed = next((i for i in range(last, len(rest)) if rest[i].startswith("s_waitcnt vmcnt(0)")), len(rest))
    used = next((i for i in range(last, len(rest)) if rest[i].startswith(("ds_", "global_store", "s_endpgm"))), len(rest))
    need(landed < used, "LDS is used again, or the kernel ends, before the last copies have landed")
    need(eight or any(landed < i < used for i in barriers(rest)), "LDS is used again before every wavefront's last copies have landed")
    return len(body)


def check_mx_gemm_distances(name: str, fn: list) -> int:
    """The wait states around instructions from assembly, which the compiler does not insert.  Two between a vector instruction that writes an operand
    (fragment, scale, sum) of a scaled matrix instruction and that one; 24 (16 passes and what a vector instruction needs behind them, with some to
    spare) between it and any other access to its sums; five between a vector instruction that writes scalar registers (a lane's read, a comparison)
    and a copy that takes its descriptor or offset from these.  On every way through the code; an instruction counts as one state, s_nop n as n + 1.
    Returns the number of instructions that were checked; raises on a violation."""
    import re
    two_results = ("v_swap", "v_permlane16_swap", "v_permlane32_swap")
    scalar_results = ("v_cmp", "v_readlane", "v_readfirstlane", "v_add_co", "v_addc", "v_sub_co", "v_subb", "v_subrev_co", "v_mad_u64", "v_mad_i64", "v_div_scale")

    def registers(operand):
        out = set()
        for kind, lo, hi, one in re.findall(r"\b([vas])\[(\d+):(\d+)\]|\b([vas]\d+)\b", operand):
            out |= {one} if one else {f"{kind}{i}" for i in range(int(lo), int(hi) + 1)}
        return out

    class Instruction:
        def __init__(self, line):
            self.op, _, args = line.partition(" ")
            # (modifiers name no registers)
            args = [x.strip() for x in re.split(r",(?![^\[]*\])", args)] if args else []
            self.uses = [registers(x) for x in args]
            self.states = int(args[0], 0) + 1 if self.op == "s_nop" else 1
            vector = self.op.startswith("v_") and not self.op.startswith("v_mfma")
            self.wrote = set().union(*self.uses[:2 if self.op.startswith(two_results) else 1]) if vector else set()
            self.wrote_scalars = {r for u in self.uses[:2] for r in u if r[0] == "s"} if self.op.startswith(scalar_results) else set()
            self.target = args[0] if re.match(r"s_c?branch", self.op) else None
            self.before, self.behind = [], []

    code, labels = [], {}
    for line in (l.split(";")[0].strip() for l in fn):
        if m := re.match(r"^([.\w]+):", line):
            labels[m.group(1)] = len(code)
        elif line and not line.startswith("."):
            code.append(Instruction(line))
    for i, x in enumerate(code):
        if x.op not in ("s_branch", "s_endpgm") and i + 1 < len(code):
            x.behind.append(i + 1)
        if x.target is not None:
            x.behind.append(labels[x.target])
        for j in x.behind:
            code[j].before.append(i)

    def look(i, states, way, hit, what):
        left, todo = {}, [(j, states) for j in getattr(code[i], way)]
        while todo:
            j, n = todo.pop()
            if n <= left.get(j, 0):
                continue
            left[j] = n
            if hit(code[j]):
                raise RuntimeError(f"{name}: {what}: {code[j].op}")
            todo += [(k, n - code[j].states) for k in getattr(code[j], way)]

    checked = 0
    for i, x in enumerate(code):
        if x.op.startswith("v_mfma_scale"):
            operands, sums = set().union(*x.uses[:6]), x.uses[0]
            look(i, 2, "before", lambda c: bool(c.wrote & operands), "an operand of a matrix instruction is written within two wait states before it")
            look(i, 24, "behind", lambda c: not c.op.startswith("v_mfma") and any(sums & u for u in c.uses), "a sum is used too close behind its matrix instruction")
            checked += 1
        elif x.op.startswith("buffer_load"):
            scalars = {r for u in x.uses for r in u if r[0] == "s"}
            look(i, 5, "before", lambda c: bool(c.wrote_scalars & scalars), "a copy's scalar registers are written within five wait states before it")
            checked += 1
    return checked


EXT_PKG = ROOT / "dhellam"
EXT_SUFFIX = sysconfig.get_config_var("EXT_SUFFIX")
PY_INCLUDE = sysconfig.get_paths()["include"]


def torch_extension_path() -> Path:
    return EXT_PKG / ("_Clib" + EXT_SUFFIX)


def host_extension_path() -> Path:
    return PKG / ("_host" + EXT_SUFFIX)


def _build_extension(src: Path, out: Path, rpath: str, verbose: bool) -> Path:
    """Host code only: the host compiler with torch's headers, linked against ``libdhellam_hip.so`` (found at run
    time relative to the extension)."""
    import torch
    from torch.utils import cpp_extension as E
    if not LIB_PATH.exists():
        raise RuntimeError(f"{LIB_PATH} must be built first")
    rocm = Path(os.environ.get("ROCM_PATH", "/opt/rocm"))
    name = out.name.split(".")[0]
    tmp = out.with_suffix(".so.tmp")
    torch_lib = E.library_paths()[0]
    cmd = [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-Wno-unused-function",
           "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", f"-DTORCH_EXTENSION_NAME={name}", "-DTORCH_API_INCLUDE_EXTENSION_H",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f"-I{ROOT / 'include'}", *[f"-isystem{p}" for p in E.include_paths()], f"-isystem{rocm / 'include'}",
           f"-I{PY_INCLUDE}", str(src), "-o", str(tmp),
           f"-L{torch_lib}", "-lc10", "-lc10_hip", "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python", "-lamdhip64",
           f"-L{LIB_DIR}", "-ldhellam_hip", f"-Wl,-rpath,{rpath}", f"-Wl,-rpath,{torch_lib}"]
    if verbose:
        print(" ".join(cmd), flush=True)
    res = subprocess.run(cmd, capture_output=True, text=True)
    if res.returncode != 0:
        raise RuntimeError(f"building {name} failed:\n{res.stderr}")
    if res.stderr.strip() and verbose:
        print(res.stderr, file=sys.stderr)
    os.replace(tmp, out)
    return out


def build_torch_extension(verbose: bool = False) -> Path:
    """Compiles ``csrc/torchapi.cpp`` into the pybind11 torch extension ``dhellam._Clib`` (the reference builds a
    module of that name from its csrc/torchapi.cpp, setup.py:234-244)."""
    return _build_extension(CSRC / "torchapi.cpp", torch_extension_path(), "$ORIGIN/../dhellam_amd/lib", verbose)


def build_host_extension(verbose: bool = False) -> Path:
    """Compiles ``csrc/hostapi.cpp`` into ``dhellam_amd._host``, the host path of the Python operators."""
    return _build_extension(CSRC / "hostapi.cpp", host_extension_path(), "$ORIGIN/lib", verbose)


def build_extensions(verbose: bool = False) -> list[Path]:
    """Both extensions, side by side."""
    with ThreadPoolExecutor(max_workers=2) as ex:
        return [f.result() for f in [ex.submit(build_host_extension, verbose), ex.submit(build_torch_extension, verbose)]]


if __name__ == "__main__":
    path = build(verbose="-v" in sys.argv)
    print(path)
    print(f"grouped GEMM main loops checked: {check_grouped_gemm_loops(verbose='-v' in sys.argv)}")
    print(f"microscaled GEMM main loops checked: {check_mx_gemm_loops(verbose='-v' in sys.argv)}")
    if "--no-ext" not in sys.argv:
        for path in build_extensions(verbose="-v" in sys.argv):
            print(path)
