"""Builds and loads `_cs_torch` (csrc/torch_ops.cpp), the extension on torch's
C++ tensors.  Like `_cs_fast` it is a speed-up of the host path: without it
the same entry points are reached from Python."""
from __future__ import annotations

import os
import subprocess
import sysconfig
import warnings

from . import fastcall

HERE = fastcall.HERE
MODULE = "_cs_torch"
SOURCE = os.path.join(HERE, "csrc", "torch_ops.cpp")


def build(lib_path: str, verbose: bool = False) -> str:
    """Compiles the module next to the library it links (rpath $ORIGIN)."""
    import torch
    from torch.utils import cpp_extension
    # A module from an earlier build must not outlive a failed one.
    for f in os.listdir(HERE):
        if f.startswith(MODULE) and f.endswith(".so"):
            os.remove(os.path.join(HERE, f))
    out = os.path.join(HERE, MODULE + sysconfig.get_config_var("EXT_SUFFIX"))
    tmp = out + ".tmp"
    libdir, libfile = os.path.split(lib_path)
    torch_lib = os.path.join(os.path.dirname(torch.__file__), "lib")
    includes = [*cpp_extension.include_paths(), os.path.join(fastcall.ROCM, "include"),
                sysconfig.get_paths()["include"]]
    cmd = ["g++", "-O2", "-shared", "-fPIC", "-std=c++17", "-Wall", "-Werror",
           "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM",
           f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
           f'-DCS_SIGNATURE_HASH="{fastcall.signature_hash()}"',
           *[a for i in includes for a in ("-isystem", i)], "-o", tmp, SOURCE,
           "-L", libdir, "-l:" + libfile, "-L", torch_lib, "-ltorch_python", "-ltorch_cpu",
           "-lc10", "-lc10_hip", "-Wl,-rpath,$ORIGIN"]
    if verbose:
        print(" ".join(cmd), flush=True)
    subprocess.check_call(cmd)
    os.replace(tmp, out)
    return out


_MODULE = False   # not looked up yet


def module():
    """The extension, or None when it has not been built."""
    global _MODULE
    if _MODULE is False:
        from . import _native as N
        N.lib()   # the library that the extension links, by the path it was built at
        try:
            from . import _cs_torch
        except ImportError:
            _cs_torch = None
        if _cs_torch is not None and _cs_torch.signature_hash() != fastcall.signature_hash():
            warnings.warn("repo_amd._cs_torch was built from other entry-point signatures; "
                          "it is not used (run build() again)")
            _cs_torch = None
        _MODULE = _cs_torch
    return _MODULE
