"""Build libpocketlm_hip.so in-tree with hipcc for gfx950.

    python -m pocketlm_amd.build            # compile every .hip source, link
    python -m pocketlm_amd.build --jobs 8

Each source under csrc/ is compiled to an object in csrc/_build/ (in
parallel), then linked into pocketlm_amd/libpocketlm_hip.so.  Only the
symbols declared in include/pocketlm_hip.h are exported.

Where a kernel needs more vector registers than it has, hipcc can save one at
the end of a divergent region before it enables the other lanes again, which
then read back what was in memory before.  Such a kernel faults now and then, so
the build reads each source's assembly and fails at such a store
(masked_spills).
"""

from __future__ import annotations

import argparse
import os
import re
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

PKG_DIR = Path(__file__).resolve().parent
REPO_DIR = PKG_DIR.parent
CSRC = PKG_DIR / "csrc"
BUILD_DIR = CSRC / "_build"
LIB_PATH = PKG_DIR / "libpocketlm_hip.so"
ARCH = "gfx950"

COMMON_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-fvisibility=hidden",
    # fp32 denormals are kept (the reference's CPU arithmetic keeps them)
    "-fno-gpu-flush-denormals-to-zero",
    # no packed-fp32 instructions
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    f"-I{REPO_DIR / 'include'}",
    f"-I{CSRC}",
]


def hipcc() -> str:
    for cand in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", shutil.which("hipcc")):
        if cand and Path(cand).exists():
            return cand
    raise RuntimeError("hipcc not found (ROCm is required to build libpocketlm_hip.so)")


def sources() -> list[Path]:
    return sorted(CSRC.glob("*.hip"))


_LABEL = re.compile(r"^(?P<function>_\w+):|^(?:\.LBB|; %bb|\.Lfunc_end)")


def masked_spills(assembly: str) -> list[str]:
    """Stores of spilled vector registers in front of the instruction that ends
    their block's divergent region, as "function: store"."""
    found, function, stores = [], "", []
    for line in assembly.splitlines():
        label = _LABEL.match(line)
        if label:
            function, stores = label["function"] or function, []
        elif "saveexec" in line:
            stores = []
        elif "Spill" in line and ("scratch_store" in line or "buffer_store" in line):
            stores.append(f"{function}: {line.strip()}")
        elif stores and "s_or_b64 exec, exec," in line:
            found += stores
            stores = []
    return found


def _compile(src: Path) -> Path:
    obj = BUILD_DIR / (src.stem + ".o")
    with tempfile.TemporaryDirectory(dir=BUILD_DIR) as temps:
        held = Path(temps) / obj.name
        cmd = [hipcc(), *COMMON_FLAGS, "-save-temps=obj", "-c", str(src), "-o", str(held)]
        proc = subprocess.run(cmd, capture_output=True, text=True)
        if proc.returncode != 0:
            raise RuntimeError(f"compile failed: {' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")
        listing = Path(temps) / f"{src.stem}-hip-amdgcn-amd-amdhsa-{ARCH}.s"
        found = masked_spills(listing.read_text())
        if found:
            raise RuntimeError(f"{src.name}: registers spilled while lanes are off, use fewer:\n" + "\n".join(found))
        os.replace(held, obj)
    return obj


def build(jobs: int | None = None, verbose: bool = False) -> Path:
    BUILD_DIR.mkdir(parents=True, exist_ok=True)
    srcs = sources()
    jobs = jobs or min(8, max(1, os.cpu_count() or 1))
    with ThreadPoolExecutor(max_workers=jobs) as pool:
        objs = list(pool.map(_compile, srcs))
    tmp = LIB_PATH.with_suffix(".so.tmp")
    cmd = [hipcc(), f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", str(tmp), *map(str, objs)]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"link failed: {' '.join(cmd)}\n{proc.stdout}\n{proc.stderr}")
    os.replace(tmp, LIB_PATH)
    if verbose:
        print(f"built {LIB_PATH} from {len(srcs)} sources")
    return LIB_PATH


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--jobs", type=int, default=None)
    args = ap.parse_args(argv)
    build(args.jobs, verbose=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())
