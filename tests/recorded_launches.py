"""Calls of the library in a process of their own whose launches are written down instead of started, as on a device of 256 CUs: which kernels a call takes, with
what grids, and what it asks for their LDS.  Runs without a GPU; operands are addresses that nothing reads."""
import json
import os
import re
import shutil
import subprocess
import sys
import tempfile

import pytest

from kutacc_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT = 1 << 40  # an address that nothing reads, aligned

RUNTIME = r"""
#include <stddef.h>
#include <stdint.h>
#include <stdio.h>
typedef struct { uint32_t x, y, z; } dim3;
static struct { const void *host; const char *name; } kernels[4096];
static int count;
static dim3 grid_, block_;
static size_t lds_;
static const char *name_of(const void *host)
{
    for (int i = 0; i < count; ++i) {
        if (kernels[i].host == host) return kernels[i].name;
    }
    return "?";
}
void **__hipRegisterFatBinary(const void *data) { static void *handle; return &handle; }
void __hipUnregisterFatBinary(void **modules) {}
void __hipRegisterVar(void **m, void *v, char *h, char *n, int e, size_t s, int c, int g) {}
void __hipRegisterFunction(void **m, const void *host, char *device, const char *name, unsigned t, void *a, void *b, void *c, void *d, int *w)
{
    if (count < 4096) kernels[count].host = host, kernels[count++].name = name;
}
int hipGetDevice(int *d) { *d = 0; return 0; }
int hipDeviceGetAttribute(int *v, int which, int d) { *v = 256; return 0; }
int hipGetLastError(void) { return 0; }
int hipFuncSetAttribute(const void *f, int which, int v) { printf("lds %s %d\n", name_of(f), v); fflush(stdout); return 0; }
unsigned __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, void *stream) { grid_ = grid, block_ = block, lds_ = lds; return 0; }
int __hipPopCallConfiguration(dim3 *grid, dim3 *block, size_t *lds, void **stream) { *grid = grid_, *block = block_, *lds = lds_, *stream = 0; return 0; }
int hipLaunchKernel(const void *f, dim3 grid, dim3 block, void **args, size_t lds, void *stream)
{
    printf("launch %s %u %u %u %u %zu\n", name_of(f), grid.x, grid.y, grid.z, block.x, lds);
    fflush(stdout);
    return 0;
}
"""

CALLS = """
import ctypes, json, sys
sys.modules["torch"] = None  # or it would bring a runtime of its own
ctypes.CDLL(sys.argv[1], ctypes.RTLD_GLOBAL)  # in front of the runtime that the library brings
sys.path.insert(0, sys.argv[2])
from kutacc_amd import capi
for function, struct, fields in json.load(open(sys.argv[3])):
    print("call", flush=True)
    if struct:
        args = getattr(capi, struct)()
        for k, v in fields.items():
            setattr(args, k, v)
        rc = getattr(capi.lib(), function)(ctypes.byref(args), None)
    else:
        rc = getattr(capi.lib(), function)(*fields, None)
    print("rc", rc, flush=True)
"""


class Launch:
    def __init__(self, name, x, y, z, threads, lds):
        self.kernel = name
        self.grid, self.threads, self.lds = (int(x), int(y), int(z)), int(threads), int(lds)

    def __repr__(self):
        return f"{self.kernel} {self.grid} x {self.threads}, {self.lds} bytes"


class Record:
    """Of one call: its code, its launches in order, and the dynamic LDS that kernels were opted into, as (kernel, bytes)."""

    def __init__(self, text):
        self.rc = int(re.search(r"^rc (-?\d+)$", text, re.M).group(1))
        self.launches = [Launch(*m) for m in re.findall(r"^launch (\S+) (\d+) (\d+) (\d+) (\d+) (\d+)$", text, re.M)]
        self.opted = [(name, int(n)) for name, n in re.findall(r"^lds (\S+) (\d+)$", text, re.M)]

    def __repr__(self):
        return f"rc {self.rc}: {self.launches}"


def record(calls):
    """One Record for each of `calls`: (function, name of its argument structure in capi, fields), or (function, None, arguments but the stream)."""
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None or not os.path.exists(build.LIB_PATH):
        pytest.skip("needs the built library and a C compiler")
    with tempfile.TemporaryDirectory() as tmp:
        source, shim, asked = (os.path.join(tmp, n) for n in ("runtime.c", "runtime.so", "calls.json"))
        with open(source, "w") as f:
            f.write(RUNTIME)
        with open(asked, "w") as f:
            json.dump(calls, f)
        subprocess.run([cc, "-shared", "-fPIC", "-O1", "-w", source, "-o", shim], check=True)
        out = subprocess.run([sys.executable, "-c", CALLS, shim, ROOT, asked], capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-2000:]
    texts = out.stdout.split("call\n")[1:]
    assert len(texts) == len(calls), out.stdout[-2000:]
    return [Record(t) for t in texts]
