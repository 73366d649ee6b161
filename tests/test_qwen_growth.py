"""A prefill whose larger buffers cannot be had leaves a decoder that makes them again, or says so, and never
launches on buffers that are gone.  On the CPU: a stand-in for the HIP runtime, loaded ahead of it, counts
allocations and launches, refuses allocations when told to, and runs nothing.  As the runtime does, it keeps the
thread's last error until it is asked for, which is how launches are checked."""
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
PKG = Path(__file__).resolve().parent.parent / "index-tts-25-metal_amd"

# Device memory is host memory that nothing touches; copies and kernels do nothing.
STAND_IN = r"""
#include <cstddef>
#include <cstdint>
#include <cstdlib>
struct Dim { uint32_t x, y, z; };
extern "C" {
int allocations = 0, launches = 0, refuse_from = 0, last = 0;  // refuse_from: the first allocation that fails, 0 for none
int hipMalloc(void** p, size_t n) {
    *p = ++allocations >= refuse_from && refuse_from ? nullptr : std::malloc(n);
    return *p ? 0 : (last = 2);
}
int hipFree(void* p) { std::free(p); return 0; }
int hipHostMalloc(void** p, size_t n, unsigned) { *p = std::calloc(1, n); return 0; }
int hipHostFree(void* p) { std::free(p); return 0; }
int hipMemcpy(void*, const void*, size_t, int) { return 0; }
int hipMemcpyAsync(void*, const void*, size_t, int, void*) { return 0; }
int hipMemsetAsync(void*, int, size_t, void*) { return 0; }
int hipStreamCreateWithFlags(void** s, unsigned) { *s = &launches; return 0; }
int hipStreamDestroy(void*) { return 0; }
int hipStreamSynchronize(void*) { return 0; }
int hipDeviceSynchronize() { return 0; }
int hipEventCreate(void** e) { *e = &launches; return 0; }
int hipEventCreateWithFlags(void** e, unsigned) { *e = &launches; return 0; }
int hipEventDestroy(void*) { return 0; }
int hipEventRecord(void*, void*) { return 0; }
int hipEventSynchronize(void*) { return 0; }
int hipGetDevice(int* d) { *d = 0; return 0; }
int hipDeviceGetAttribute(int* v, int, int) { *v = 256; return 0; }
int hipGetLastError() {
    const int e = last;
    last = 0;
    return e;
}
int __hipPushCallConfiguration(Dim, Dim, size_t, void*) { return 0; }
int __hipPopCallConfiguration(Dim* g, Dim* b, size_t* l, void** s) {
    *g = *b = Dim{1, 1, 1};
    *l = 0;
    *s = nullptr;
    return 0;
}
int hipLaunchKernel(const void*, Dim, Dim, void**, size_t, void*) { return ++launches, 0; }
}
"""

SCRIPT = r"""
import ctypes, sys
hip = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
import numpy as np
import itts_gpt as it

def value(name):
    return ctypes.c_int.in_dll(hip, name)

shapes = {"qwen.model.embed_tokens.weight": (151936, 1024), "qwen.model.norm.weight": (1024,)}
for name, shape in (("self_attn.q_proj", (2048, 1024)), ("self_attn.k_proj", (1024, 1024)), ("self_attn.v_proj", (1024, 1024)),
                    ("self_attn.o_proj", (1024, 2048)), ("self_attn.q_norm", (128,)), ("self_attn.k_norm", (128,)),
                    ("mlp.gate_proj", (3072, 1024)), ("mlp.up_proj", (3072, 1024)), ("mlp.down_proj", (1024, 3072)),
                    ("input_layernorm", (1024,)), ("post_attention_layernorm", (1024,))):
    shapes[f"qwen.model.layers.0.{name}.weight"] = shape
weights = {k: np.zeros(v, np.float32) for k, v in shapes.items()}  # (pages that are never written take no memory)
made = value("allocations")
for bits in (32, 4):
    d = it.QwenDecoder(weights, layers=1, weight_bits=bits)
    before = made.value
    d.prefill([1] * 300)
    first = made.value - before
    d.prefill([1] * 20)
    assert first >= 6 and made.value == before + first and value("launches").value > 0
    for nth in range(1, first + 1):
        before = made.value
        value("refuse_from").value = before + nth
        try:
            # (the workspace of the split products is made once, whatever the length)
            d.prefill([1] * (300 + 100 * nth))
            assert bits == 32 and nth == first, (bits, nth)
            value("refuse_from").value = 0
            continue
        except it.GptRuntimeError:
            pass
        launched = value("launches").value
        try:
            d.prefill([1] * 20)  # fits the buffers that were there before
            raise SystemExit(f"{bits} bits, allocation {nth}: a prefill without its buffers")
        except it.GptRuntimeError:
            pass
        assert value("launches").value == launched, (bits, nth)
        value("refuse_from").value = 0
        d.prefill([1] * 20)
        assert value("launches").value > launched
    d.close()
print("fine")
"""


def test_a_failed_growth_leaves_no_missing_buffers(tmp_path):
    source, lib = tmp_path / "stand_in.cpp", tmp_path / "stand_in.so"
    source.write_text(STAND_IN)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-o", str(lib), str(source)], check=True)
    p = subprocess.run([sys.executable, "-c", SCRIPT, str(lib)], cwd=PKG, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.strip() == "fine", p.stdout + p.stderr[-2000:]
