"""Host-only runs of the library: a stand-in for the HIP runtime's calls that keeps
a list of the kernels launched and runs none. It is loaded into a child process
ahead of the library, so that the library's calls bind to it."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = r"""
#include <stddef.h>
#include <string.h>
typedef struct { unsigned x, y, z; } dim3_t;
enum { MAX = 8192 };
static const void *key[MAX];
static const char *name[MAX];
static int n_key, n_call, fail, last, device, set; /* last: as hipGetLastError gives it */
static const char *call[MAX];
static dim3_t grid, block;
static size_t shared;
static void *stream;

void **__hipRegisterFatBinary(const void *d) { static void *h; return &h; }
void __hipUnregisterFatBinary(void **m) {}
void __hipRegisterVar(void **m, void *v, char *h, char *d, int e, size_t s, int c, int g) {}
void __hipRegisterFunction(void **m, const void *host, char *dev, const char *dname, unsigned t,
                           void *a, void *b, void *c, void *d, int *w) {
    if (n_key < MAX && strstr(dname, "9rsllm_hip")) { key[n_key] = host; name[n_key++] = dname; }
}
static const char *find(const void *f) {
    for (int i = 0; i < n_key; i++) if (key[i] == f) return name[i];
    return "?";
}
int __hipPushCallConfiguration(dim3_t g, dim3_t b, size_t l, void *s) {
    grid = g; block = b; shared = l; stream = s; return 0;
}
int __hipPopCallConfiguration(dim3_t *g, dim3_t *b, size_t *l, void **s) {
    *g = grid; *b = block; *l = shared; *s = stream; return 0;
}
int hipLaunchKernel(const void *f, dim3_t g, dim3_t b, void **a, size_t l, void *s) {
    if (n_call < MAX) call[n_call++] = find(f);
    return 0;
}
int hipFuncSetAttribute(const void *f, int attr, int value) {
    if (fail > 0) { fail--; return last = 2; } /* hipErrorOutOfMemory */
    set++;
    return 0;
}
int hipGetDevice(int *d) { *d = device; return 0; }
int hipSetDevice(int d) { device = d; return 0; }
int hipGetDeviceCount(int *n) { *n = 2; return 0; }
int hipStreamCreateWithFlags(void **s, unsigned f) { *s = &device; return 0; }
int hipStreamDestroy(void *s) { return 0; }
int hipGetSymbolAddress(void **p, const void *s) { *p = &device; return 0; }
int hipGetLastError(void) { int e = last; last = 0; return e; }

void rec_fail(int n) { fail = n; } /* the next n hipFuncSetAttribute */
int rec_set(void) { int n = set; set = 0; return n; } /* hipFuncSetAttribute granted since */
int rec_kernels(void) { return n_key; }
const char *rec_kernel(int i) { return name[i]; }
const char *rec_take(void) { return n_call ? call[--n_call] : ""; } /* the last one */
"""

PRELUDE = """
import ctypes, sys
rec = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
rec.rec_kernel.restype = rec.rec_take.restype = ctypes.c_char_p
from rsllm_amd import backend as B
assert rec.rec_kernels() > 0, "the library did not bind to the stand-in"
"""


def run(folder, code):
    """What `code` (with the binding as B and the stand-in as rec) prints."""
    src, lib = os.path.join(folder, "rec.c"), os.path.join(folder, "librec.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-o", lib, src], check=True)
    r = subprocess.run([sys.executable, "-c", PRELUDE + code, lib], cwd=ROOT, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]
    return r.stdout
