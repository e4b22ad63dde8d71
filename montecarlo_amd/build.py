"""Build libmi355mc.so (the C-ABI + HIP kernels) in-tree with hipcc for gfx950.

hipcc cross-compiles without a GPU; the library is git-ignored and stays in
the tree beside its sources.  Usage:  python -m montecarlo_amd.build [--force] [--sanitize]
(--sanitize: the host-only sources under ASan + UBSan into libmi355mc_host_san.so, see build_sanitized)
"""
from __future__ import annotations

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libmi355mc.so")
SOURCES = ["mc_table.cpp", "mc_train.cpp", "mc_ingest.cpp", "mc_device.hip", "mc_rank.hip", "mc_sort.hip", "mc_runs.hip", "mc_gn.hip", "mc_enum.hip", "mc_logits_score.hip",
           "mc_logits_gradient.hip", "mc_logits_draw.hip", "mc_comm.cpp"]
HEADERS = [os.path.join(CSRC, "mc_internal.h"), os.path.join(CSRC, "mc_sort.h"), os.path.join(CSRC, "mc_philox.h"),
           os.path.join(CSRC, "mc_logits.h"),
           os.path.join(os.path.dirname(HERE), "include", "mi355mc.h")]
# (packed float32 instructions stay off: some of their forms have given wrong results on this hardware; the host pass
# does not know the feature and would say so for every file)
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-ffp-contract=off", "-Wall", "-Wno-unused-function",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
LINK_FLAGS = ["--offload-arch=gfx950", "-shared", "-fPIC", "-ldl"]


def sources_digest() -> str:
    """sha256 over the native sources the library is built from (names and bytes) and the flags it is built with: a
    measurement of the kernels (profiles/hbm_traffic_latest.json) records it, and bench.py quotes the measurement only while
    it still holds."""
    import hashlib
    h = hashlib.sha256("\n".join(FLAGS + LINK_FLAGS).encode())
    for path in sorted([os.path.join(CSRC, s) for s in SOURCES] + HEADERS):
        h.update(os.path.basename(path).encode())
        with open(path, "rb") as f:
            h.update(f.read())
    return h.hexdigest()


def needs_build() -> bool:
    if not os.path.exists(LIB):
        return True
    t = os.path.getmtime(LIB)
    deps = [os.path.join(CSRC, s) for s in SOURCES] + HEADERS + [os.path.abspath(__file__)]      # (the flags stand here)
    return any(os.path.getmtime(d) > t for d in deps)


HOST_SOURCES = ["mc_table.cpp", "mc_train.cpp", "mc_ingest.cpp"]       # no GPU code: table compiler, trainers, ingest, writers
HOST_SAN_LIB = os.path.join(HERE, "libmi355mc_host_san.so")
SAN_FLAGS = ["-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer", "-fsanitize=address,undefined",
             "-fno-sanitize-recover=undefined", "-fPIC", "-shared", "-ffp-contract=off", "-pthread", "-Wall",
             "-Wno-unused-function"]


def sanitizer_runtime() -> str:
    """Path of the AddressSanitizer runtime g++ links against ('' when the image has none): a process that loads the
    sanitized library without being built with the sanitizer itself (python) preloads it (LD_PRELOAD)."""
    gxx = os.environ.get("CXX", "g++")
    try:
        path = subprocess.run([gxx, "-print-file-name=libasan.so"], capture_output=True, text=True, check=True).stdout.strip()
    except (OSError, subprocess.CalledProcessError):
        return ""
    return os.path.realpath(path) if os.path.isabs(path) and os.path.exists(path) else ""


def build_sanitized(force: bool = False, verbose: bool = True) -> str:
    """The host-only part of the library (everything that parses caller-supplied text and dict shapes) under
    AddressSanitizer + UndefinedBehaviorSanitizer, for tests/test_sanitized_host.py.  CPU code only: nothing here
    touches the GPU."""
    deps = [os.path.join(CSRC, s) for s in HOST_SOURCES] + HEADERS
    if not force and os.path.exists(HOST_SAN_LIB) and all(os.path.getmtime(d) <= os.path.getmtime(HOST_SAN_LIB) for d in deps):
        return HOST_SAN_LIB
    if not sanitizer_runtime():
        raise RuntimeError("no AddressSanitizer runtime in this image (g++ -print-file-name=libasan.so)")
    cmd = [os.environ.get("CXX", "g++")] + SAN_FLAGS + ["-o", HOST_SAN_LIB] + [os.path.join(CSRC, s) for s in HOST_SOURCES]
    if verbose:
        print(" ".join(cmd), file=sys.stderr)
    subprocess.run(cmd, check=True)
    return HOST_SAN_LIB


def build(force: bool = False, verbose: bool = True) -> str:
    if not force and not needs_build():
        return LIB
    import tempfile
    from concurrent.futures import ThreadPoolExecutor
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    with tempfile.TemporaryDirectory(prefix="mi355mc_") as tmp:
        objects = [os.path.join(tmp, s + ".o") for s in SOURCES]

        def compile_one(job):
            cmd = [hipcc] + FLAGS + ["-c", "-o", job[1], os.path.join(CSRC, job[0])]
            if verbose:
                print(" ".join(cmd), file=sys.stderr)
            done = subprocess.run(cmd, stderr=subprocess.PIPE, text=True)
            said = [ln for ln in done.stderr.splitlines() if "'-packed-fp32-ops' is not a recognized feature" not in ln]
            if said:
                print("\n".join(said), file=sys.stderr)
            if done.returncode:
                raise subprocess.CalledProcessError(done.returncode, cmd)

        with ThreadPoolExecutor(min(8, len(SOURCES))) as pool:
            list(pool.map(compile_one, zip(SOURCES, objects)))
        cmd = [hipcc] + LINK_FLAGS + ["-o", LIB + ".new"] + objects
        if verbose:
            print(" ".join(cmd), file=sys.stderr)
        subprocess.run(cmd, check=True)
        os.replace(LIB + ".new", LIB)          # (a process that has the old library mapped keeps its own)
    return LIB


if __name__ == "__main__":
    if "--sanitize" in sys.argv:
        print(build_sanitized(force="--force" in sys.argv))
    else:
        build(force="--force" in sys.argv)
