"""The compiled binding of the dense site's operators (csrc/torch_binding.cpp): torch tensors in and out,
checks, allocations, streams and autograd rules in C++ above the C ABI.  Loaded on first use; there is no
fallback, a missing build raises with the build command."""
from __future__ import annotations

import importlib.util
import os

from . import _lib

MODULE_PATH = os.path.join(_lib.PKG, "_mortar_native.so")


class _Native:
    def loaded(self) -> bool:
        return "_module" in self.__dict__

    def __getattr__(self, name):
        if not self.loaded():
            _lib.lib()                                         # the library it is linked against, and its error if missing
            if not os.path.exists(MODULE_PATH):
                raise ImportError(f"{MODULE_PATH} is missing: the extension must be built first "
                                  f"(python {os.path.join(_lib.PKG, 'build.py')}); there is no fallback")
            spec = importlib.util.spec_from_file_location("_mortar_native", MODULE_PATH)
            module = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(module)
            self.__dict__["_module"] = module
        value = getattr(self.__dict__["_module"], name)
        self.__dict__[name] = value                            # later look-ups find the function at once
        return value


native = _Native()
