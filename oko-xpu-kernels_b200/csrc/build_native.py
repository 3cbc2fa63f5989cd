"""Compiles the torch binding (binding.cpp) beside the package: build_native.py SOURCE OUTPUT."""

import os
import subprocess
import sys
import sysconfig

import torch
from torch.utils import cpp_extension

source, output = sys.argv[1:3]
root = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
cuda = os.environ.get("CUDA_HOME", "/usr/local/cuda")
includes = [os.path.join(root, "include"), sysconfig.get_paths()["include"], os.path.join(cuda, "include"),
            *cpp_extension.include_paths()]
libraries = os.path.join(os.path.dirname(torch.__file__), "lib")
# The C++ runtime that torch has loaded, by its path and before the compiler's own: a compiler that finds
# only a static one would give the module a second runtime, whose streams (the messages of torch's
# checks) crash beside the first.
with open("/proc/self/maps") as maps:
    runtime = sorted({line.split()[-1] for line in maps if "/libstdc++.so" in line})
subprocess.run([os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden",
                f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
                *dict.fromkeys("-isystem" + i if i != includes[0] else "-I" + i for i in includes),
                source, "-o", output, *runtime, "-L" + libraries, "-ltorch_python", "-ltorch", "-ltorch_cpu", "-ltorch_cuda",
                "-lc10", "-lc10_cuda", "-Wl,-rpath," + libraries], check=True)
