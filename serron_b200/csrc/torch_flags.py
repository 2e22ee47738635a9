"""Prints the compiler flags of an extension for the installed torch: include paths, ABI and libraries."""

import sysconfig

import torch
from torch.utils import cpp_extension

flags = [f"-isystem {p}" for p in [*cpp_extension.include_paths("cuda"), sysconfig.get_paths()["include"]]]
flags.append(f"-D_GLIBCXX_USE_CXX11_ABI={int(torch.compiled_with_cxx11_abi())}")
flags += [f"-L{p}" for p in cpp_extension.library_paths()]
flags += ["-lc10", "-lc10_cuda", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
print(" ".join(flags))
