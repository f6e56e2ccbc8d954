"""Build recipe for libltkv.so (HIP kernels + host block manager, gfx950).

Run as ``python -m langtrain_studio_amd.build``. Cross-compiles without a GPU.
"""

from __future__ import annotations

import os
import shlex
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

PKG = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(PKG, "csrc")
LIB = os.path.join(PKG, "libltkv.so")
# The profiling build: the same sources with -DLTKV_TIMELINE (per-wave phase
# stamps of the decode kernel, ltkv_timeline_read), for bench.py's timeline
# workloads; the product never loads it.
TIMELINE_LIB = os.path.join(PKG, "libltkv_timeline.so")
SOURCES = [os.path.join(CSRC, "ltkv_cache.cpp"), os.path.join(CSRC, "ltkv_kernels.hip"),
           os.path.join(CSRC, "ltkv_scored.hip"), os.path.join(CSRC, "ltkv_scored_rows.hip"),
           os.path.join(CSRC, "ltkv_scored_chunk.hip")]
HEADERS = [os.path.join(CSRC, "ltkv_kernels.h"), os.path.join(CSRC, "ltkv_device.h"),
           os.path.join(CSRC, "ltkv_scored.h"), os.path.join(os.path.dirname(PKG), "include", "ltkv.h")]

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
ARCH = "gfx950"
# Packed FP32 (v_pk_*_f32) is disabled for all device code. MFMA operands and
# results live in VGPRs: with AGPR accumulators the decode attention kernel
# copied its 32 accumulators between AGPRs and VGPRs on every tile.
DEVICE_FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", "-mllvm", "-amdgpu-mfma-vgpr-form"]
COMMON = ["-O3", "-std=c++17", "-fPIC", "-fvisibility=hidden", "-Wall", "-Wno-unused-command-line-argument"]


VERSION_SCRIPT = os.path.join(CSRC, "ltkv.map")


def compile_command(source: str, obj: str, timeline: bool) -> list[str]:
    return [HIPCC, f"--offload-arch={ARCH}", *COMMON, *DEVICE_FLAGS, *(["-DLTKV_TIMELINE"] if timeline else []),
            "-c", source, "-o", obj]


def link_command(objects: list[str], out: str) -> list[str]:
    return [HIPCC, f"--offload-arch={ARCH}", "-shared", "-fPIC", f"-Wl,--version-script={VERSION_SCRIPT}", "-o", out,
            *objects]


def run(cmd: list[str], verbose: bool) -> str:
    """Runs a compiler command; an error text, or nothing."""
    if verbose:
        print("+", " ".join(shlex.quote(c) for c in cmd), flush=True)
    proc = subprocess.run(cmd, stderr=subprocess.PIPE, stdout=subprocess.DEVNULL, text=True)
    # hipcc's host pass warns that it does not know the packed-fp32 feature: harmless.
    noise = ("packed-fp32-ops", "not a recognized feature", "warning: unknown target feature")
    err = "\n".join(l for l in proc.stderr.splitlines() if not any(n in l for n in noise))
    if proc.returncode != 0:
        return f"hipcc failed ({proc.returncode}) for {os.path.basename(cmd[-1])}:\n{err}"
    if verbose and err.strip():
        print(err, file=sys.stderr)
    return ""


def build(verbose: bool = True, timeline: bool = True) -> str:
    """Compile every source into libltkv.so (always recompiles), and the
    profiling build libltkv_timeline.so beside it: every source by itself, as
    many at a time as there are processors (at most 8). Sources without phase
    stamps serve both libraries."""
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
        objects: dict[bool, list[str]] = {False: [], True: []}
        jobs = []
        for source in sorted(SOURCES, key=os.path.getsize, reverse=True):  # the longest first
            with open(source) as f:
                stamped = "LTKV_TIMELINE" in f.read()
            for tl in (False, True) if stamped and timeline else (False,):
                obj = os.path.join(tmp, os.path.basename(source) + (".timeline.o" if tl else ".o"))
                jobs.append(pool.submit(run, compile_command(source, obj, tl), verbose))
                objects[tl].append(obj)
                if not stamped:
                    objects[True].append(obj)
        failed = [e for e in (job.result() for job in jobs) if e]
        for tl in (False, True) if timeline else (False,):
            out = TIMELINE_LIB if tl else LIB
            if not failed and (e := run(link_command(objects[tl], out + ".tmp"), verbose)):
                failed.append(e)
        if failed:
            raise RuntimeError("\n".join(failed))
        for tl in (False, True) if timeline else (False,):
            out = TIMELINE_LIB if tl else LIB
            os.replace(out + ".tmp", out)
    return LIB


if __name__ == "__main__":
    build(timeline="--no-timeline" not in sys.argv[1:])
