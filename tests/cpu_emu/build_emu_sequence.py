"""TEST INFRASTRUCTURE: compiles the kernel sources of the sequence products for the CPU against tests/cpu_emu/hip_emu.h
(tests/cpu_emu/_build/libf3m_sequence_emu.so, never loaded by the f3m_amd package)."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
CSRC = os.path.join(ROOT, "f3m_amd", "csrc")
OUT = os.path.join(HERE, "_build", "libf3m_sequence_emu.so")
SRCS = ["f3m_attention.hip", "f3m_linear.hip"]


def build(force=False):
    srcs = [os.path.join(CSRC, s) for s in SRCS]
    deps = srcs + [os.path.join(CSRC, h) for h in ("f3m_rt.h", "f3m_tile.h")] + \
        [os.path.join(HERE, "hip_emu.h"), os.path.join(ROOT, "include", "f3m_sequence.h"), os.path.abspath(__file__)]
    if not force and os.path.exists(OUT) and all(os.path.getmtime(OUT) > os.path.getmtime(p) for p in deps):
        return OUT
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    # the engine's f3m_last_error lives in a source that this library leaves out
    last = os.path.join(HERE, "_build", "sequence_last_error.cpp")
    with open(last, "w") as f:
        f.write('#include "f3m_rt.h"\nextern "C" const char *f3m_last_error(void) { return f3m::g_error.c_str(); }\n')
    flags = ["-O1", "-g", "-fPIC", "-std=c++17", "-DF3M_CPU_EMU", "-I", HERE, "-I", CSRC, "-I", os.path.join(ROOT, "include"), "-Wall",
             "-Wno-unused", "-Wno-unknown-pragmas", "-Wno-maybe-uninitialized"]
    objs, jobs = [], []
    for s in srcs + [last]:
        o = os.path.join(HERE, "_build", os.path.basename(s) + ".seq.o")
        jobs.append(subprocess.Popen(["g++"] + flags + ["-x", "c++", "-c", s, "-o", o]))
        objs.append(o)
    for j in jobs:
        if j.wait():
            raise RuntimeError("g++ failed")
    subprocess.check_call(["g++", "-shared", "-o", OUT] + objs)
    return OUT


if __name__ == "__main__":
    print(build(force=True))
