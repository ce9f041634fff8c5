"""The runtime's argument checks (csrc/runtime/group_args.h) built for the
host, so that what a launch accepts is tested without a GPU."""
import ctypes
import os
import subprocess

import hfusion_mi355x as hf
from hfusion_mi355x import native

SOURCE = r"""
#include "group_args.h"
#include <chrono>
#include <fstream>
static std::string why;
extern "C" {
GroupArgs *args_load(const char *manifest) {
  auto *g = new GroupArgs();
  std::ifstream f(manifest);
  for (std::string ln; std::getline(f, ln);) {
    std::istringstream is(ln);
    std::string key;
    is >> key;
    if (key == "func") is >> g->func;
    else if (key == "rows_dyn") g->rowsDyn = true;
    else g->line(key, is);
    if (is.fail() && !ln.empty()) { delete g; return nullptr; }
  }
  if (!g->prepare()) { delete g; return nullptr; }
  return g;
}
void args_free(GroupArgs *g) { delete g; }
const char *args_check(const GroupArgs *g, const uint64_t *p, size_t n, void *const *r, size_t nr, int64_t rows) {
  why = g->check(p, n, r, nr, rows);
  return why.c_str();
}
const char *args_workspace(const GroupArgs *g, uint64_t at) {
  why = g->checkWorkspace((const void *)(uintptr_t)at);
  return why.c_str();
}
// ns of a check that passes, the best of 200 runs of 1000
double args_time(const GroupArgs *g, const uint64_t *p, size_t n, void *const *r, size_t nr, int64_t rows) {
  double best = 1e30;
  for (int i = 0; i < 200; ++i) {
    const auto t = std::chrono::steady_clock::now();
    size_t bad = 0;
    for (int k = 0; k < 1000; ++k) bad += !g->check(p, n, r, nr, rows).empty();
    const double ns = std::chrono::duration<double, std::nano>(std::chrono::steady_clock::now() - t).count() / 1000;
    if (bad) return -1;
    best = ns < best ? ns : best;
  }
  return best;
}
}
"""
_lib = None


def lib(folder):
    global _lib
    if _lib is None:
        src, so = os.path.join(folder, "args.cpp"), os.path.join(folder, "args.so")
        with open(src, "w") as f:
            f.write(SOURCE)
        subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Wextra", "-shared", "-fPIC", "-I",
                        os.path.join(native.PKG_ROOT, "csrc", "runtime"), "-o", so, src], check=True)
        _lib = ctypes.CDLL(so)
        p = ctypes.c_void_p
        call = [p, ctypes.POINTER(ctypes.c_uint64), ctypes.c_size_t, ctypes.POINTER(p), ctypes.c_size_t, ctypes.c_int64]
        _lib.args_load.argtypes, _lib.args_load.restype = [ctypes.c_char_p], p
        _lib.args_free.argtypes = [p]
        _lib.args_check.argtypes, _lib.args_check.restype = call, ctypes.c_char_p
        _lib.args_workspace.argtypes, _lib.args_workspace.restype = [p, ctypes.c_uint64], ctypes.c_char_p
        _lib.args_time.argtypes, _lib.args_time.restype = call, ctypes.c_double
    return _lib


_BYTES = {"f64": 8, "i64": 8, "index": 8, "f32": 4, "i32": 4, "f16": 2, "bf16": 2, "i16": 2}


class Checked:
    """A group's checks; `at`, `res`: addresses that do not overlap."""

    def __init__(self, ir, folder, options="", rows=-1):
        art = hf.compile(ir, options=options)
        self.lib, self.meta, self.rows = lib(str(folder)), art.blocks[0], rows
        self.h = self.lib.args_load(art.manifest.encode())
        assert self.h
        where, step = 1 << 40, 1 << 32
        assert all(self.bytes(b) < step // 2 for k in ("params", "results") for b in self.meta[k])
        self.at, self.res = [], []
        for kind, out in (("params", self.at), ("results", self.res)):
            for b in self.meta[kind]:
                out.append(where if b.get("tied", -1) < 0 else 0)
                where += step

    def __del__(self):
        if getattr(self, "h", None):
            self.lib.args_free(self.h)

    def bytes(self, b):
        n = _BYTES.get(b["elem"], 1)
        for d in b["shape"]:
            n *= self.rows if d < 0 else d
        return n

    def param_bytes(self, i):
        return self.bytes(self.meta["params"][i])

    def result_bytes(self, i):
        return self.bytes(self.meta["results"][i])

    def _packed(self, at, res):
        a, r = list(self.at), list(self.res)
        for i, v in (at or {}).items():
            a[i] = v
        for i, v in (res or {}).items():
            r[i] = v
        return (self.h, (ctypes.c_uint64 * max(1, len(a)))(*a), len(a), (ctypes.c_void_p * max(1, len(r)))(*r), len(r), self.rows)

    def why(self, at=None, res=None):
        """What a launch says with these addresses in place of its own."""
        return self.lib.args_check(*self._packed(at, res)).decode()

    def why_workspace(self, at):
        return self.lib.args_workspace(self.h, at).decode()

    def ns(self):
        return self.lib.args_time(*self._packed(None, None))
