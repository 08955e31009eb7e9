"""The paged cache's operators on the CPU: refusals, and the index arithmetic that keeps what comes from
device memory inside the tensors (compiled here as plain C++ from the header the kernels use)."""
import ctypes
import random
import subprocess

import pytest

torch = pytest.importorskip("torch")

import kvcache_oracle as ref  # noqa: E402
from kernel_anvil import _native, kvcache  # noqa: E402
from kernel_anvil._native import ANVIL_ERR_ALIGN, ANVIL_ERR_INVALID, ANVIL_ERR_UNSUPPORTED, AnvilError  # noqa: E402

SHIM = """
#include "kv_index.h"
extern "C" void seq(int a, int b, int kv, int total, long long cap, int *o) {
    anvil::KvSeq s = anvil::kv_seq(a, b, kv, total, cap);
    o[0] = s.q0; o[1] = s.q1; o[2] = s.kv; o[3] = s.bad;
}
extern "C" long long row(int page, int pages, int head, int heads, int off, int shift) {
    return anvil::kv_row(page, pages, head, heads, off, shift);
}
extern "C" int seen(int i, int n, int kv, int causal) { return anvil::kv_seen(i, n, kv, causal); }
"""
EDGES = [-2 ** 31, -2 ** 31 + 1, -1, 0, 1, 2, 63, 64, 1000, 2 ** 31 - 2, 2 ** 31 - 1]


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_index")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(_native.CSRC), "-o", str(d / "shim.so"),
                    str(d / "shim.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "shim.so"))
    lib.row.restype = ctypes.c_longlong
    lib.seq.argtypes = [ctypes.c_int] * 4 + [ctypes.c_longlong, ctypes.c_void_p]
    return lib


def test_starts_and_lengths_stay_in_range(index):
    o = (ctypes.c_int * 4)()
    for total in (0, 1, 64, 2 ** 31 - 1):
        for cap in (0, 16, 2 ** 31 - 1):
            for a in EDGES:
                for b in EDGES:
                    for kv in EDGES:
                        index.seq(a, b, kv, total, cap, o)
                        q0, q1, n, bad = o
                        assert 0 <= q0 <= q1 <= total and 0 <= n <= cap
                        assert bool(bad) == ((q0, q1, n) != (a, b, kv))


def test_rows_stay_in_the_cache_beyond_32_bits(index):
    rng = random.Random(1)
    for _ in range(2000):
        shift, heads = rng.randint(0, 10), rng.randint(1, 64)
        pages = rng.choice([1, 7, 2 ** 20, 2 ** 31 - 1])
        head, off = rng.randrange(heads), rng.randrange(1 << shift)
        for page in EDGES + [pages - 1, pages, rng.randrange(pages)]:
            got = index.row(ctypes.c_int(page), pages, head, heads, off, shift)
            if 0 <= page < pages and page <= 2 ** 31 - 1:
                assert got == (page * heads + head) * (1 << shift) + off
            else:
                assert got == -1


def test_rows_see_the_tokens_up_to_their_own(index):
    for n, kv in ((1, 0), (1, 1), (4, 10), (10, 4), (3, 3), (2 ** 30, 2 ** 31 - 1)):
        for i in {0, min(1, n - 1), n // 2, n - 1}:
            assert index.seen(i, n, kv, 0) == kv
            assert index.seen(i, n, kv, 1) == max(0, min(kv, kv - n + i + 1))


# ---- the C ABI's refusals: nothing is launched, so no GPU is needed --------------------------

def c_cache(**kw):
    a = dict(kind=8, num_pages=4, kv_heads=2, page_size=16, head_dim=128, k=4096, v=8192, k_scale=16, v_scale=32)
    a.update(kw)
    return kvcache._Cache(**a)


def c_batch(**kw):
    a = dict(page_table=64, page_table_stride=4, max_pages=4, batch=2, total=3, start=128, kv_len=256)
    a.update(kw)
    return kvcache._Batch(**a)


CACHE_FAULTS = [
    (dict(kind=3), ANVIL_ERR_UNSUPPORTED), (dict(kind=0), ANVIL_ERR_UNSUPPORTED),
    (dict(head_dim=96), ANVIL_ERR_UNSUPPORTED), (dict(head_dim=0), ANVIL_ERR_UNSUPPORTED),
    (dict(page_size=0), ANVIL_ERR_INVALID), (dict(page_size=24), ANVIL_ERR_INVALID),
    (dict(page_size=2048), ANVIL_ERR_INVALID), (dict(num_pages=0), ANVIL_ERR_INVALID),
    (dict(kv_heads=0), ANVIL_ERR_INVALID), (dict(kv_heads=70000), ANVIL_ERR_INVALID),
    (dict(k=None), ANVIL_ERR_INVALID), (dict(v_scale=None), ANVIL_ERR_INVALID),
    (dict(v=8200), ANVIL_ERR_ALIGN), (dict(k_scale=20), ANVIL_ERR_ALIGN),
]
BATCH_FAULTS = [
    (dict(batch=-1), ANVIL_ERR_INVALID), (dict(total=-1), ANVIL_ERR_INVALID), (dict(max_pages=-1), ANVIL_ERR_INVALID),
    (dict(page_table_stride=3), ANVIL_ERR_INVALID), (dict(start=None), ANVIL_ERR_INVALID),
    (dict(page_table=None), ANVIL_ERR_INVALID), (dict(start=130), ANVIL_ERR_ALIGN), (dict(kv_len=258), ANVIL_ERR_ALIGN),
]


def calls(c, b, k=16, v=32, dtype=1, stride=256, heads=4, out=64, work=16, nbytes=1 << 40):
    lib, c, b = _native.lib(), ctypes.byref(c), ctypes.byref(b)
    return {"write": lambda: lib.anvil_kv_write(c, b, dtype, k, stride, 128, v, stride, 128, None),
            "read": lambda: lib.anvil_kv_read(c, b, None, dtype, k, v, None),
            "attention": lambda: lib.anvil_paged_attention(c, b, dtype, k, stride, 128, heads, 1.0, 1, out, work, nbytes,
                                                           None)}


@pytest.mark.parametrize("fault,status", CACHE_FAULTS + BATCH_FAULTS, ids=lambda x: str(x))
def test_c_abi_refuses_bad_caches_and_batches(fault, status):
    in_cache = any(f is fault for f, _ in CACHE_FAULTS)
    c, b = (c_cache(**fault), c_batch()) if in_cache else (c_cache(), c_batch(**fault))
    for name, call in calls(c, b).items():
        assert call() == status, name
        assert _native.last_error()
    assert _native.lib().anvil_paged_attention_workspace(ctypes.byref(c), ctypes.byref(b), 4) == status


@pytest.mark.parametrize("which,kw,status", [
    ("write", dict(dtype=2), ANVIL_ERR_UNSUPPORTED), ("read", dict(dtype=8), ANVIL_ERR_UNSUPPORTED),
    ("attention", dict(dtype=0), ANVIL_ERR_UNSUPPORTED), ("write", dict(k=None), ANVIL_ERR_INVALID),
    ("read", dict(v=None), ANVIL_ERR_INVALID), ("attention", dict(k=None), ANVIL_ERR_INVALID),
    ("attention", dict(out=None), ANVIL_ERR_INVALID), ("attention", dict(heads=3), ANVIL_ERR_INVALID),
    ("attention", dict(heads=0), ANVIL_ERR_INVALID), ("write", dict(k=18), ANVIL_ERR_ALIGN),
    ("write", dict(stride=255), ANVIL_ERR_ALIGN), ("read", dict(k=24), ANVIL_ERR_ALIGN),
    ("attention", dict(stride=260), ANVIL_ERR_ALIGN), ("attention", dict(out=68), ANVIL_ERR_ALIGN),
])
def test_c_abi_refuses_bad_arguments(which, kw, status):
    assert calls(c_cache(), c_batch(), **kw)[which]() == status


def test_c_abi_refuses_null_structs_and_mixed_types():
    lib = _native.lib()
    assert lib.anvil_kv_read(None, None, None, 1, 16, 16, None) == ANVIL_ERR_INVALID
    assert lib.anvil_paged_attention_workspace(None, None, 4) == ANVIL_ERR_INVALID
    for kind, dtype in ((1, 30), (30, 1)):
        c = c_cache(kind=kind, k_scale=None, v_scale=None)
        assert calls(c, c_batch(), dtype=dtype)["attention"]() == ANVIL_ERR_UNSUPPORTED
    assert calls(c_cache(), c_batch(kv_len=None))["write"]() == ANVIL_ERR_INVALID
    assert calls(c_cache(), c_batch(kv_len=None))["attention"]() == ANVIL_ERR_INVALID


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 2.9e38, -3.4e38])
def test_c_abi_refuses_scales_that_are_not_finite(scale):
    """2.9e38 is finite, but not times log2(e), which the scores are multiplied by."""
    status = _native.lib().anvil_paged_attention(ctypes.byref(c_cache()), ctypes.byref(c_batch()), 1, 16, 256, 128, 4,
                                                 scale, 1, 64, 32, 1 << 40, None)
    assert status == ANVIL_ERR_INVALID and "scale" in _native.last_error()


def test_c_abi_empty_calls_do_nothing():
    for b in (c_batch(total=0, start=None, page_table=None), c_batch(batch=0)):
        for name, call in calls(c_cache(), b, k=None, v=None, out=None).items():
            assert call() == 0, name


def test_c_abi_flags():
    """Unknown ones are refused; with ANVIL_FLAG_ZERO_REST a batch of no sequences has rows to write."""
    lib, zero = _native.lib(), _native.ANVIL_FLAG_ZERO_REST
    read = lambda b, flags, dtype=1, k=16, v=32: lib.anvil_kv_read_ex(  # noqa: E731
        ctypes.byref(c_cache()), ctypes.byref(b), None, dtype, k, v, flags, None)
    attention = lambda b, flags, out=64: lib.anvil_paged_attention_ex(  # noqa: E731
        ctypes.byref(c_cache()), ctypes.byref(b), 1, 16, 256, 128, 4, 1.0, 1, out, 32, 1 << 40, flags, None)
    for flags in (1, 4, 1 << 31, zero | 1):
        assert read(c_batch(), flags) == ANVIL_ERR_INVALID and "flags" in _native.last_error()
        assert attention(c_batch(), flags) == ANVIL_ERR_INVALID and "flags" in _native.last_error()
    nobody = c_batch(batch=0)
    assert read(nobody, 0, k=None) == 0 and attention(nobody, 0, out=None) == 0
    assert read(nobody, zero, k=None) == read(nobody, zero, v=None) == attention(nobody, zero, out=None) == ANVIL_ERR_INVALID
    assert read(nobody, zero, dtype=2) == ANVIL_ERR_UNSUPPORTED
    assert read(c_batch(batch=0, total=0), zero, k=None) == attention(c_batch(batch=0, total=0), zero, out=None) == 0


# ---- the Python surface ------------------------------------------------------------------------

def test_cache_shapes_and_refusals():
    for kind, last in (("F16", 128), ("BF16", 128), ("Q8_0", 128), ("Q4_0", 64)):
        c = kvcache.PagedKVCache(5, 16, 2, 128, kind, device="cpu")
        assert c.k.shape == (5, 2, 16, last)
        assert c.bytes_per_token == 2 * 2 * {"F16": 256, "BF16": 256, "Q8_0": 136, "Q4_0": 72}[kind]
    for args in ((5, 16, 2, 96), (5, 24, 2, 128), (5, 2048, 2, 128), (0, 16, 2, 128), (5, 16, 0, 128)):
        with pytest.raises(AnvilError):
            kvcache.PagedKVCache(*args, device="cpu")
    with pytest.raises(AnvilError):
        kvcache.PagedKVCache(5, 16, 2, 128, "Q5_0", device="cpu")
    t = torch.zeros(5, 2, 16, 128, dtype=torch.int8)
    s = torch.zeros(5, 2, 16, 4, dtype=torch.float16)
    for bad in ((t, t, None, s), (t, t, s, s.float()), (t, t[:4], s, s), (t, t.half(), s, s), (t[0], t[0], s, s),
                (t, t, s, s[..., :2])):
        with pytest.raises(AnvilError):
            kvcache.PagedKVCache.from_buffers("Q8_0", *bad)
    with pytest.raises(AnvilError):
        kvcache.PagedKVCache.from_buffers("F16", t.half(), t.half(), s, s)


def test_no_cpu_path():
    batch = ref.Batch("Q8_0", 64, 2, 16, [3], [20])
    cache = kvcache.PagedKVCache.from_buffers("Q8_0", batch.k, batch.v, batch.ks, batch.vs)
    x = torch.randn(3, 2, 64)
    for call in (lambda: kvcache.kv_write(cache, x, x, batch.table, batch.start, batch.kv_len),
                 lambda: kvcache.kv_read(cache, batch.table, batch.start, 3),
                 lambda: kvcache.paged_attention(x.half(), cache, batch.table, batch.start, batch.kv_len)):
        with pytest.raises(AnvilError, match="no CPU path"):
            call()


def test_the_module_needs_nothing_of_a_torch_with_cuda_to_be_imported():
    """A torch built without CUDA lacks torch._C's CUDA functions: the import still works, and calls are refused."""
    import os
    import sys

    code = """
import torch
for name in [n for n in dir(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
from kernel_anvil import kvcache
cache = kvcache.PagedKVCache(5, 16, 2, 128, "F16", device="cpu")
table, start = torch.zeros(1, 5, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32)
try:
    kvcache.kv_read(cache, table, start, 3)
except kvcache.AnvilError as e:
    assert "no CPU path" in str(e)
else:
    raise SystemExit(1)
"""
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    subprocess.run([sys.executable, "-c", code], check=True, env=env, timeout=300)


def test_inputs_of_either_differentiation_are_refused():
    """Neither a gradient nor a tangent is dropped silently (refused before anything else, so no GPU is needed)."""
    from torch.autograd import forward_ad

    batch = ref.Batch("F16", 64, 2, 16, [3], [20])
    cache = kvcache.PagedKVCache.from_buffers("F16", batch.k, batch.v)
    args = (batch.table, batch.start, batch.kv_len)
    x = torch.randn(3, 2, 64).half()
    with pytest.raises(AnvilError, match="backward"):
        kvcache.paged_attention(x.clone().requires_grad_(), cache, *args)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: kvcache.paged_attention(dual, cache, *args), lambda: kvcache.kv_write(cache, dual, x, *args),
                     lambda: kvcache.kv_write(cache, x, dual, *args)):
            with pytest.raises(AnvilError, match="forward-mode"):
                call()
        with pytest.raises(AnvilError, match="no CPU path"):    # others pass this check
            kvcache.paged_attention(x, cache, *args)
    with torch.no_grad(), pytest.raises(AnvilError, match="no CPU path"):
        kvcache.paged_attention(x.clone().requires_grad_(), cache, *args)


def test_rules_are_the_gguf_types():
    """Codes and scales of the oracle (which the GPU tests hold the kernels to) against gguf-py's blocks:
    equal but where a value stands within fp32 rounding of a border."""
    import numpy as np
    from gguf import GGMLQuantizationType as T
    from gguf import quants

    x = torch.randn(400, 128, generator=torch.Generator().manual_seed(0))
    for kind, t, nb in (("Q8_0", T.Q8_0, 34), ("Q4_0", T.Q4_0, 18)):
        blocks = quants.quantize(x.numpy(), t).reshape(400, 4, nb)
        codes, scales = ref.quantise(kind, x)
        d = torch.from_numpy(np.ascontiguousarray(blocks[..., :2]).view(np.float16)[..., 0].copy())
        same = (d == scales).float().mean()
        assert same > 0.999 and ((d.float() - scales.float()).abs() <= 2.0 ** -10 * d.float().abs()).all()
        got = torch.from_numpy(blocks[..., 2:].copy().reshape(codes.shape).view(np.int8 if kind == "Q8_0" else np.uint8))
        assert (got == codes).float().mean() > 0.9995
