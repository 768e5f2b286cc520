"""Build libmsf2.so in-tree with hipcc for gfx950 (cross-compiles without a GPU)."""
import hashlib
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
HEADER = os.path.join(os.path.dirname(HERE), "include", "msf2.h")
# translation unit -> the headers it includes; the units are compiled side by side and linked into one library
UNITS = {
    "msf2_api.hip": ("msf2_common.h", "msf2_gemm.h", "msf2_gemm_bf16.h", "msf2_gemm_bf16_astat.h", "msf2_attn_fused.h",
                     "msf2_linkv_bf16.h", "msf2_ops.h"),
    "msf2_blocks.hip": ("msf2_common.h", "msf2_rows.h", "msf2_groupnorm.h", "msf2_recurrence.h", "msf2_dropout.h"),
}
# Packed fp32 arithmetic stays off: hipcc makes v_pk_add/mul/fma_f32 of ordinary float code by itself, and some of their
# forms have given wrong results on this hardware now and then.  (The host pass warns that it does not know the feature.)
FLAGS = ["-O3", "--offload-arch=gfx950", "-std=c++17", "-fPIC", "-Wno-unused-value", "-Wno-inline-asm",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
OUT = os.path.join(HERE, "lib", "libmsf2.so")


STAMP = OUT + ".sources.sha256"


def _digest(files) -> str:
    h = hashlib.sha256()
    for d in files:
        with open(d, "rb") as f:
            h.update(os.path.basename(d).encode() + b"\0" + f.read())
    h.update(" ".join(FLAGS).encode() + os.environ.get("MSF2_CXXFLAGS", "").encode())
    return h.hexdigest()


def _unit_files(unit):
    return [os.path.join(CSRC, f) for f in (unit, *UNITS[unit])] + [HEADER]


def sources_digest() -> str:
    """SHA-256 over the sources the library is built from (and the flags): the library is rebuilt whenever this
    differs from the digest recorded beside it, whatever the files' time stamps say (a fresh clone, a checkout)."""
    return _digest([f for unit in UNITS for f in _unit_files(unit)])


def up_to_date() -> bool:
    try:
        with open(STAMP) as f:
            return os.path.exists(OUT) and f.read().strip() == sources_digest()
    except OSError:
        return False


def _compile(unit, force, verbose):
    """Start the compilation of one unit; None if its object is the one that these sources give."""
    obj = os.path.join(os.path.dirname(OUT), unit + ".o")
    digest = _digest(_unit_files(unit))
    try:
        with open(obj + ".sha256") as f:
            if not force and os.path.exists(obj) and f.read().strip() == digest:
                return obj, digest, None
    except OSError:
        pass
    cmd = [os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *os.environ.get("MSF2_CXXFLAGS", "").split(), *FLAGS,
           "-c", os.path.join(CSRC, unit), "-o", obj]
    if verbose:
        cmd.insert(1, "-Rpass-analysis=kernel-resource-usage")
    return obj, digest, subprocess.Popen(cmd)


def build(force: bool = False, verbose: bool = False) -> str:
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    if not force and up_to_date():
        return OUT
    units = [_compile(unit, force, verbose) for unit in UNITS]
    codes = [p.wait() if p is not None else 0 for _, _, p in units]
    if any(codes):
        raise RuntimeError(f"hipcc failed on {[u for u, c in zip(UNITS, codes) if c]}")
    for obj, digest, p in units:
        if p is not None:
            with open(obj + ".sha256", "w") as f:
                f.write(digest + "\n")
    subprocess.run([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-shared", "-fPIC",
                    *[obj for obj, _, _ in units], "-o", OUT], check=True)
    with open(STAMP, "w") as f:
        f.write(sources_digest() + "\n")
    return OUT


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
