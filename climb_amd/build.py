"""Build the C-ABI HIP library in-tree:  python -m climb_amd.build

hipcc cross-compiles for gfx950 without a GPU.  The .so stays next to the sources (git-ignored, but it travels to
the GPU box with the snapshot)."""
from __future__ import annotations

import os
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "csrc")
LIB = os.path.join(CSRC, "libclimb_hip.so")
LIB_F16 = os.path.join(CSRC, "libclimb_hip_f16.so")      # the same sources with IEEE-half operands (common.h: CLIMB_H16_F16)
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32 (hipcc -O3 forms them from ordinary float code): some of their forms give wrong results now and then on gfx950,
# with no error.  It costs 2.5 % of the bf16 training step at 64 sequences (10.49 against 10.23 ms, twice each in turn on one box)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-fno-gpu-rdc", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


# per-source flags; and sources compiled a second time under another object name (A/B builds of one kernel inside one library)
SRC_FLAGS = {}
TWICE = {"gemm_bf16_nt4.hip": ("gemm_bf16_nt4_slp", ["-DNT4_SLP_BUILD"])}      # (17 = 2 / 5: the r04 window boundary, kept as the A/B partner of r05's)


def sources():
    return sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


def units():
    """(source, object stem, extra flags)"""
    out = []
    for s in sources():
        out.append((s, s[:-4], SRC_FLAGS.get(s, [])))
        if s in TWICE:
            out.append((s, TWICE[s][0], TWICE[s][1]))
    return out


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _made_by(record) -> str:
    """what a product was made with ("" if none is on record): other flags make another object of the same source.  Without the tree's place: a copied tree is as fresh
    as the original"""
    try:
        with open(record) as f:
            return f.read()
    except OSError:
        return ""


def _text(cmd) -> str:
    return " ".join(cmd).replace(CSRC + os.sep, "")


def _run(cmd, record, what, verbose):
    if verbose:
        print(" ".join(cmd), flush=True)
    if os.path.exists(record):
        os.remove(record)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"{what}:\n{r.stdout}\n{r.stderr}")
    with open(record, "w") as f:
        f.write(_text(cmd))


def build_library(force: bool = False, verbose: bool = True) -> str:
    _build(LIB_F16, os.path.join(CSRC, "build", "f16"), ["-DCLIMB_H16_F16=1"], force, verbose)
    return _build(LIB, os.path.join(CSRC, "build"), [], force, verbose)


def _build(LIB: str, objdir: str, extra, force: bool, verbose: bool) -> str:
    hdrs = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".h")]
    os.makedirs(objdir, exist_ok=True)
    jobs = []
    for s, stem, fl in units():
        src = os.path.join(CSRC, s)
        obj = os.path.join(objdir, stem + ".o")
        cmd = [HIPCC] + FLAGS + extra + fl + ["-c", src, "-o", obj]
        if force or _stale(obj, [src] + hdrs) or _made_by(obj + ".cmd") != _text(cmd):
            jobs.append((cmd, obj + ".cmd", f"hipcc failed on {src}"))

    with ThreadPoolExecutor(max_workers=min(8, max(1, len(jobs)))) as ex:
        list(ex.map(lambda job: _run(*job, verbose), jobs))
    objs = [os.path.join(objdir, stem + ".o") for _, stem, _ in units()]
    cmd, record = [HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs, os.path.join(objdir, "link.cmd")
    if force or jobs or _stale(LIB, objs) or _made_by(record) != _text(cmd):
        _run(cmd, record, "link failed", verbose)
    return LIB


if __name__ == "__main__":
    print(build_library(force="--force" in sys.argv))
