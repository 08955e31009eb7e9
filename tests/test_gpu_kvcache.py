"""The paged cache's write, read and attention on the GPU against their definitions in 64 bits.

Bars: write and read are exact (codes, scales and rounded values bit for bit); the attention is within the
bound that kvcache_oracle.attention derives from the roundings a kernel may make.
"""
import pytest

torch = pytest.importorskip("torch")

import kvcache_oracle as ref  # noqa: E402
from kernel_anvil import kvcache as ops  # noqa: E402
from kernel_anvil import mmvq  # noqa: E402
from kernel_anvil._native import AnvilError  # noqa: E402

pytestmark = pytest.mark.gpu

KINDS = ["F16", "BF16", "Q8_0", "Q4_0"]


def q_types(kind):
    return {"F16": ["f16"], "BF16": ["bf16"]}.get(kind, ["f16", "bf16"])


KIND_TYPES = [(k, t) for k in KINDS for t in q_types(k)]


def make_q(batch, heads, dtype, extra=0, pad=0, amp=1.0):
    """q (rows + extra, heads, dim) inside wider rows when pad > 0."""
    x = amp * torch.randn(batch.rows + extra, heads + pad, batch.dim, generator=batch.gen)
    return x.to(ref.NP[dtype]).cuda()[:, pad // 2:pad // 2 + heads]


def check_attention(batch, heads, dtype, causal=True, scale=None, pad=0, amp=1.0, q=None):
    q = make_q(batch, heads, dtype, pad=pad, amp=amp) if q is None else q
    table, start, kv_len = batch.on_gpu()
    got = ops.paged_attention(q, batch.cache(ops), table, start, kv_len, scale=scale, causal=causal)
    torch.cuda.synchronize()
    want, tol = ref.attention(batch, q.cpu(), batch.dim ** -0.5 if scale is None else scale, causal)
    got = got.cpu().double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine)
    over = ((got - want).abs() - tol)[fine]
    assert over.numel() == 0 or over.max() <= 0, \
        f"worst excess {over.max():.3e}, largest error {((got - want).abs())[fine].max():.3e}"
    assert mmvq.take_device_status() == 0
    return got


# ---- write and read ----------------------------------------------------------------------

def nasty(x):
    """Rows with zeros, ties, equal magnitudes, tiny and huge values and values beside the borders."""
    f = x.view(-1, 32)
    f[0] = 0
    f[1] = torch.arange(32) - 15.5                        # halves of the step once the block's top is 127 / 2
    f[1, 0] = 63.5
    f[2] = torch.linspace(-127, 127, 32)
    f[3] = 2.0 * (torch.arange(32) % 2) - 1               # equal magnitudes, negative first
    f[4] = 1 - 2.0 * (torch.arange(32) % 2)               # equal magnitudes, positive first
    f[5] = 1e-30 * torch.arange(32)
    f[6] = (torch.arange(32) - 16) / 2                    # halves of Q4_0's step
    f[7] *= 1e-6
    f[8] = 3.0e4
    f[9] = (torch.arange(32) + 0.5) * (8.0 / 8)
    f[9, 5] = -127
    return x


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_write_is_exact(kind, dim, dtype):
    q_lens, past = [5, 0, 1, 33, 17], [0, 9, 31, 70, 3]
    batch = ref.Batch(kind, dim, 3, 16, q_lens, [a + b for a, b in zip(q_lens, past)], seed=dim, wide=2)
    x = [nasty(torch.randn(batch.rows + 2, 3, dim, generator=batch.gen)) for _ in range(2)]
    k, v = (t.to(ref.NP[dtype]) for t in x)
    cache = batch.cache(ops)
    table, start, kv_len = batch.on_gpu()
    before = [t.clone() for t in (cache.k, cache.v)]
    ops.kv_write(cache, k.cuda(), v.cuda(), table, start, kv_len)   # two rows behind the last sequence
    for name, new in (("k", k), ("v", v)):
        codes, scales = ref.quantise(kind, new)
        t, s = (batch.k, batch.ks) if name == "k" else (batch.v, batch.vs)
        for b, n in enumerate(q_lens):
            if n:
                p, o = batch.slots(b, torch.arange(past[b], past[b] + n))
                rows = slice(int(batch.start[b]), int(batch.start[b]) + n)
                t[p, :, o] = codes[rows]
                if s is not None:
                    s[p, :, o] = scales[rows]
        assert torch.equal(getattr(cache, name).cpu(), t), f"{name} codes"     # written rows and all others
        if s is not None:
            assert torch.equal(getattr(cache, name + "_scale").cpu(), s), f"{name} scales"
    assert not torch.equal(cache.k, before[0])
    assert mmvq.take_device_status() == 0


def test_write_decides_borders_of_fp32_values_exactly():
    """fp32 values on and one step beside the borders between two codes."""
    g = torch.Generator().manual_seed(5)
    for kind in ("Q8_0", "Q4_0"):
        M = torch.rand(4096, 1, generator=g) + 0.5
        n = torch.randint(0, 127 if kind == "Q8_0" else 8, (4096, 31), generator=g) + 0.5
        x = (n.double() * M.double() / (127 if kind == "Q8_0" else 8)).float()
        step = torch.randint(-2, 3, x.shape, generator=g).int()
        x = (x.view(torch.int32) + step).view(torch.float32) * (1 - 2 * torch.randint(0, 2, x.shape, generator=g))
        x = torch.minimum(x.abs(), M) * torch.sign(x)
        x = torch.cat([M, x], -1).view(-1, 2, 64)
        batch = ref.Batch(kind, 64, 2, 64, [x.shape[0]], [x.shape[0]])
        cache = batch.cache(ops)
        ops.kv_write(cache, x.cuda(), -x.cuda(), *batch.on_gpu())
        p, o = batch.slots(0, torch.arange(x.shape[0]))
        for t, s, new in ((cache.k, cache.k_scale, x), (cache.v, cache.v_scale, -x)):
            codes, scales = ref.quantise(kind, new)
            assert torch.equal(t.cpu()[p, :, o], codes)
            assert torch.equal(s.cpu()[p, :, o], scales)


@pytest.mark.parametrize("kind", ["Q8_0", "Q4_0"])
def test_write_saturates_and_keeps_nan_in_its_block(kind):
    x = torch.randn(4, 1, 64)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 0], x[2, 0, 33] = 1e30, float("-inf"), float("nan"), 7.0e4
    batch = ref.Batch(kind, 64, 1, 4, [4], [4])
    cache = batch.cache(ops)
    table, start, kv_len = batch.on_gpu()
    ops.kv_write(cache, x.cuda(), x.cuda(), table, start, kv_len)
    got, _ = ops.kv_read(cache, table, start, 4)
    codes, scales = ref.quantise(kind, x)
    want = ref.values(kind, codes, scales).float()
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.cpu()), torch.nan_to_num(want))
    assert torch.isnan(want[2, 0, :32]).all() and torch.isfinite(want[2, 0, 32:]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page", [(64, 1), (128, 16), (256, 8), (128, 1024)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_read_is_exact(kind, dim, page, dtype):
    lens, first = [0, 1, 37, 16, 65], [0, 4, 0, 20, 3]
    batch = ref.Batch(kind, dim, 2, page, lens, [a + b for a, b in zip(lens, first)], seed=page)
    table, start, _ = batch.on_gpu()
    got = ops.kv_read(batch.cache(ops), table, start, batch.rows, first=torch.tensor(first, dtype=torch.int32).cuda(),
                      dtype=ref.NP[dtype])
    for name, t in zip("kv", got):
        want = torch.cat([batch.rows_of(name, b)[f:] for b, f in enumerate(first)])
        assert torch.equal(t.cpu(), want.to(ref.NP[dtype]))
    assert mmvq.take_device_status() == 0


def test_read_without_first_and_into_given_buffers():
    batch = ref.Batch("Q8_0", 128, 8, 32, [40, 3], [64, 3])
    table, start, _ = batch.on_gpu()
    out = tuple(torch.full((45, 8, 128), 7.0, device="cuda") for _ in range(2))
    got = ops.kv_read(batch.cache(ops), table, start, 45, out=out)
    assert got[0] is out[0]
    want = torch.cat([batch.rows_of("k", 0, 40), batch.rows_of("k", 1, 3)]).float()
    assert torch.equal(out[0][:43].cpu(), want)
    assert (out[0][43:] == 7).all() and (out[1][43:] == 7).all()   # rows behind the last sequence


def test_strided_inputs_and_unaligned_rows_are_written():
    batch = ref.Batch("F16", 64, 2, 16, [9], [9])
    table, start, kv_len = batch.on_gpu()
    wide = torch.randn(9, 6, 65, dtype=torch.float16, device="cuda")
    for k, v in ((wide[:, 0:2, :64], wide[:, 2:4, 1:]), (wide[:, 0:4:2, :64], wide.flip(0)[:, 4:, :64])):
        cache = batch.cache(ops)
        ops.kv_write(cache, k, v, table, start, kv_len)
        rk, rv = ops.kv_read(cache, table, start, 9, dtype=torch.float16)
        assert torch.equal(rk, k) and torch.equal(rv, v)


# ---- attention ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind,dtype", KIND_TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_lens,past", [
    ([1], [0]), ([1, 1, 1], [0, 63, 200]),                  # single tokens
    ([3, 1, 5, 2], [14, 0, 129, 64]),                       # a few tokens
    ([40, 1, 129], [0, 300, 77]),                           # chunks among single tokens
    ([0, 2, 0], [5, 0, 0]),                                 # sequences without new tokens
])
def test_attention_kinds_and_lengths(kind, dtype, dim, q_lens, past):
    batch = ref.Batch(kind, dim, 2, 16, q_lens, [a + b for a, b in zip(q_lens, past)], seed=dim)
    check_attention(batch, 8, dtype)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 16, 17, 40])
@pytest.mark.parametrize("q_lens", [[1, 1], [2, 9], [70, 3]])
def test_attention_head_groups(group, q_lens):
    batch = ref.Batch("Q8_0", 128, 2, 32, q_lens, [90, 150], seed=group)
    check_attention(batch, 2 * group, "bf16")


@pytest.mark.parametrize("page", [1, 2, 16, 64, 128, 512, 1024])
@pytest.mark.parametrize("kind,dtype", [("Q4_0", "f16"), ("BF16", "bf16")])
def test_attention_page_sizes(page, kind, dtype):
    batch = ref.Batch(kind, 64, 1, page, [1, 20, 4], [700, 131, 4], seed=page, wide=3)
    check_attention(batch, 4, dtype)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kind,dtype,dim", [("F16", "f16", 128), ("Q8_0", "bf16", 64), ("BF16", "bf16", 256)])
def test_attention_both_masks(causal, kind, dtype, dim):
    batch = ref.Batch(kind, dim, 2, 16, [150, 1, 260, 6], [150, 80, 300, 6], seed=3)
    check_attention(batch, 6, dtype, causal=causal)


@pytest.mark.parametrize("kv", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_attention_lengths_around_tiles(kv):
    for kind, dtype, dim in (("Q8_0", "f16", 128), ("BF16", "bf16", 64)):
        batch = ref.Batch(kind, dim, 1, 8, [1, min(kv, 30)], [kv, kv], seed=kv)
        check_attention(batch, 8, dtype)


@pytest.mark.parametrize("rows", [15, 16, 17, 32, 33, 127, 128, 129, 255, 256, 257, 300])
def test_attention_rows_around_tiles(rows):
    for kind, dtype, dim in (("Q4_0", "bf16", 128), ("F16", "f16", 256)):
        batch = ref.Batch(kind, dim, 1, 32, [rows], [rows + 5], seed=rows)
        check_attention(batch, 1, dtype)
        check_attention(batch, 3, dtype, causal=False)


@pytest.mark.parametrize("dim,dtype,kind", [(128, "bf16", "Q8_0"), (64, "f16", "Q4_0"), (256, "f16", "F16")])
def test_attention_long_contexts(dim, dtype, kind):
    """One sequence split over the whole card, beside short ones."""
    batch = ref.Batch(kind, dim, 2, 64, [1, 1, 5], [20011, 3, 9000], seed=dim)
    check_attention(batch, 8, dtype)
    batch = ref.Batch(kind, dim, 1, 256, [70], [15001], seed=dim)
    check_attention(batch, 4, dtype)


def test_attention_many_sequences():
    lens = [(37 * i) % 210 for i in range(300)]
    q = [(i * 7) % 3 if n > 2 else min(1, n) for i, n in enumerate(lens)]
    batch = ref.Batch("Q8_0", 64, 1, 16, q, lens, seed=9)
    check_attention(batch, 4, "bf16")


@pytest.mark.parametrize("kind,dtype", KIND_TYPES)
def test_attention_sharp_and_shifted_scores(kind, dtype):
    """Scores whose maximum grows and falls along the keys by hundreds: the running maximum moves."""
    batch = ref.Batch(kind, 128, 1, 16, [1, 90], [1000, 700], seed=4, amp=3.0)
    check_attention(batch, 4, dtype, amp=4.0)
    check_attention(batch, 4, dtype, amp=0.0)            # all scores equal
    check_attention(batch, 4, dtype, scale=0.0)
    check_attention(batch, 4, dtype, scale=-0.3)


@pytest.mark.parametrize("q_lens", [[1, 1], [9, 30], [200, 40]])
@pytest.mark.parametrize("kind,dtype", KIND_TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_attention_never_uses_what_lies_behind_the_length(q_lens, kind, dtype, value):
    batch = ref.Batch(kind, 128, 2, 64, q_lens, [201, 77], seed=1)
    batch.poison(value)
    check_attention(batch, 4, dtype)
    check_attention(batch, 4, dtype, causal=False)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("kind,dtype", KIND_TYPES)
@pytest.mark.parametrize("dim", [64, 256])
def test_a_token_reaches_only_the_rows_that_see_it(value, kind, dtype, dim):
    """Non-finite keys or values at positions that earlier rows of the chunk do not see."""
    for name in "kv":
        batch = ref.Batch(kind, dim, 1, 16, [40, 5, 150], [70, 5, 400], seed=2)
        for b, pos in ((0, 55), (1, 2), (2, 300), (2, 399)):
            batch.set_token(name, b, pos, value)
        heads = 2
        q = make_q(batch, heads, dtype)
        table, start, kv_len = batch.on_gpu()
        got = ops.paged_attention(q, batch.cache(ops), table, start, kv_len).cpu().double()
        # against the same cache with those tokens finite, for the rows before them
        clean = ref.Batch(kind, dim, 1, 16, [40, 5, 150], [70, 5, 400], seed=2)
        want, tol = ref.attention(clean, q.cpu(), dim ** -0.5, True)
        for b, pos in ((0, 55), (1, 2), (2, 300)):
            n, kv, t0 = batch.q_lens[b], batch.kv_lens[b], int(batch.start[b])
            blind = max(0, pos - (kv - n))              # rows 0 .. blind-1 stand before it
            assert ((got - want).abs() <= tol)[t0:t0 + blind].all(), (name, b)
            seeing = got[t0 + blind:t0 + n]
            if name == "v":
                assert not torch.isfinite(seeing).any(), (name, b)
            elif value != value:
                assert torch.isnan(seeing).all(), (name, b)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 3], [0, 5, 0]), ([6, 100], [2, 30]), ([300], [40]), ([1], [0])])
@pytest.mark.parametrize("kind,dtype", [("Q8_0", "bf16"), ("F16", "f16")])
def test_rows_that_see_nothing_are_zero(q_lens, kv_lens, kind, dtype):
    batch = ref.Batch(kind, 128, 2, 16, q_lens, kv_lens, wide=1)
    got = check_attention(batch, 4, dtype)
    for b, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        t0 = int(batch.start[b])
        assert (got[t0:t0 + max(0, n - kv)] == 0).all()
        if not kv:
            check = check_attention(batch, 4, dtype, causal=False)
            assert (check[t0:t0 + n] == 0).all()


@pytest.mark.parametrize("dtype,kind", [("bf16", "Q8_0"), ("f16", "F16")])
@pytest.mark.parametrize("q_lens", [[1, 1], [30, 200]])
def test_strided_queries_and_rows_behind_the_last_sequence(dtype, kind, q_lens):
    batch = ref.Batch(kind, 128, 2, 16, q_lens, [100, 250], seed=6)
    check_attention(batch, 4, dtype, pad=6)
    q = make_q(batch, 4, dtype, extra=3)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    table, start, kv_len = batch.on_gpu()
    got = ops.paged_attention(q, batch.cache(ops), table, start, kv_len, out=out)
    assert got is out and (out[batch.rows:] == 7).all()
    same = ops.paged_attention(q[:batch.rows], batch.cache(ops), table, start, kv_len)
    assert torch.equal(out[:batch.rows], same)


def test_large_queries_of_a_quantised_cache_do_not_overflow():
    """bf16 queries beyond fp16's range: scaled by a power of two, with the scores still moderate."""
    for q_lens in ([1], [100]):
        batch = ref.Batch("Q8_0", 128, 1, 16, q_lens, [300], seed=8)
        check_attention(batch, 4, "bf16", amp=1e6, scale=1e-7)
        check_attention(batch, 4, "bf16", amp=1e-9, scale=1e8)


def test_the_same_call_gives_the_same_bits():
    batch = ref.Batch("Q4_0", 128, 4, 32, [1, 1, 300, 4], [9000, 40, 2500, 900], seed=5)
    q = make_q(batch, 16, "f16")
    cache, args = batch.cache(ops), batch.on_gpu()
    a = ops.paged_attention(q, cache, *args)
    for _ in range(5):
        assert torch.equal(ops.paged_attention(q, cache, *args), a)


def test_bad_pages_and_lengths_are_cut_and_reported():
    batch = ref.Batch("Q8_0", 128, 2, 16, [2, 1], [40, 33], seed=7)
    q = make_q(batch, 4, "bf16")
    cache = batch.cache(ops)
    table, start, kv_len = batch.on_gpu()
    good = ops.paged_attention(q, cache, table, start, kv_len)
    assert mmvq.take_device_status() == 0
    for page in (-1, batch.k.shape[0], 2 ** 31 - 1):
        bad = table.clone()
        bad[1, 0] = page                                   # sequence 1 loses its first 16 tokens
        got = ops.paged_attention(q, cache, bad, start, kv_len)
        assert mmvq.take_device_status() == ops.BAD_PAGE
        assert torch.equal(got[:2], good[:2]) and torch.isfinite(got).all()
        k, v = ops.kv_read(cache, bad, torch.tensor([0, 0, 20], dtype=torch.int32).cuda(), 20)
        assert mmvq.take_device_status() == ops.BAD_PAGE
        assert (k[:16] == 0).all() and (v[:16] == 0).all() and (k[16:] != 0).any()
        before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        new = torch.randn(3, 2, 128, device="cuda")
        bad[:, 2] = page
        ops.kv_write(cache, new, new, bad, start, kv_len)
        assert mmvq.take_device_status() == ops.BAD_PAGE
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    # lengths beyond the table, negative ones, and starts out of order
    for lens in ([1000, 33], [-5, 33], [2 ** 31 - 1, 2 ** 31 - 1], [-2 ** 31, 1]):
        ops.paged_attention(q, cache, table, start, torch.tensor(lens, dtype=torch.int32).cuda())
        assert mmvq.take_device_status() == ops.BAD_PAGE
    for s in ([0, 5, 3], [-1, 2, 3], [0, 2, 99], [2 ** 31 - 1, -2 ** 31, 0]):
        ops.paged_attention(q, cache, table, torch.tensor(s, dtype=torch.int32).cuda(), kv_len)
        assert mmvq.take_device_status() == ops.BAD_PAGE
    assert torch.equal(ops.paged_attention(q, cache, table, start, kv_len), good)


def test_empty_calls():
    batch = ref.Batch("F16", 64, 1, 16, [0, 0], [5, 9])
    table, start, kv_len = batch.on_gpu()
    q = torch.empty(0, 4, 64, dtype=torch.float16, device="cuda")
    cache = batch.cache(ops)
    assert ops.paged_attention(q, cache, table, start, kv_len).shape == (0, 4, 64)
    none = torch.empty(0, 1, 64, device="cuda")
    ops.kv_write(cache, none, none, table, start, kv_len)
    assert ops.kv_read(cache, table, start, 0)[0].shape == (0, 1, 64)
    nobody = torch.zeros(1, dtype=torch.int32, device="cuda")
    table0 = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    assert ops.paged_attention(q, cache, table0, nobody, nobody[:0]).shape == (0, 4, 64)


# ---- streams, graphs, the step as a whole ----------------------------------------------------

def test_two_streams_at_once():
    """Two calls in flight on two streams keep their scratch apart."""
    jobs = []
    for i, lens in enumerate(([12000, 500], [3000, 9000])):
        batch = ref.Batch("Q8_0", 128, 2, 64, [1, 1], lens, seed=20 + i)
        jobs.append((make_q(batch, 8, "bf16"), batch.cache(ops), *batch.on_gpu()))
    want = [ops.paged_attention(*j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (j, s) in enumerate(zip(jobs, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.paged_attention(*j))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_graphs_replay_with_other_lengths_and_side_by_side():
    batch = ref.Batch("Q8_0", 128, 2, 16, [1, 3], [900, 40], seed=30)
    cache = batch.cache(ops)
    table, start, kv_len = batch.on_gpu()
    q, new = make_q(batch, 8, "bf16"), torch.randn(2, batch.rows, 2, 128, device="cuda")
    step = lambda: (ops.kv_write(cache, new[0], new[1], table, start, kv_len),  # noqa: E731
                    ops.paged_attention(q, cache, table, start, kv_len),
                    ops.kv_read(cache, table, start, batch.rows))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for lens in ([900, 40], [17, 3], [333, 35], [1, 0]):
        kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        q.normal_()
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, (torch.cuda.current_stream(), side)):  # both at once
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        want = step()
        for _, out in graphs:
            assert torch.equal(out[1], want[1])
            assert torch.equal(out[2][0], want[2][0]) and torch.equal(out[2][1], want[2][1])
    mmvq.take_device_status()   # [1, 0] has rows without a position


def test_another_stream_than_the_current_one():
    batch = ref.Batch("BF16", 64, 1, 16, [4], [50], seed=31)
    q, cache, args = make_q(batch, 2, "bf16"), batch.cache(ops), batch.on_gpu()
    want = ops.paged_attention(q, cache, *args)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = ops.paged_attention(q, cache, *args)
        torch.cuda.current_stream().synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("kind", ["Q8_0", "Q4_0", "F16"])
def test_a_decoder_layer_step_by_step_and_at_once(kind):
    """q, k, v and o products (QuantLinear) around the cache: a prompt at once, in chunks, and token by
    token leave one cache and, within rounding, one output."""
    from kernel_anvil.model import QuantLinear

    torch.manual_seed(0)
    hidden, heads, kv_heads, dim, n = 256, 4, 2, 64, 37
    mk = lambda out: QuantLinear.from_linear(torch.nn.Linear(hidden, out, bias=False).cuda())  # noqa: E731
    wq, wk, wv, wo = mk(heads * dim), mk(kv_heads * dim), mk(kv_heads * dim), \
        QuantLinear.from_linear(torch.nn.Linear(heads * dim, hidden, bias=False).cuda())
    x = torch.randn(2 * n, hidden, device="cuda", dtype=torch.float16)   # two users, n tokens each
    table = torch.tensor([[4, 1, 7], [0, 5, 2]], dtype=torch.int32, device="cuda")

    def layer(cache, rows, q_lens, kv_lens):
        start = torch.tensor([0, q_lens[0], sum(q_lens)], dtype=torch.int32, device="cuda")
        kv = torch.tensor(kv_lens, dtype=torch.int32, device="cuda")
        k, v = wk(rows).view(-1, kv_heads, dim), wv(rows).view(-1, kv_heads, dim)
        ops.kv_write(cache, k, v, table, start, kv)
        return wo(ops.paged_attention(wq(rows).view(-1, heads, dim), cache, table, start, kv).flatten(1))

    def run(cuts):
        cache = ops.PagedKVCache(9, 16, kv_heads, dim, kind)
        outs = [[], []]
        for a, b in zip(cuts, cuts[1:]):
            y = layer(cache, torch.cat([x[a:b], x[n + a:n + b]]), [b - a] * 2, [b] * 2)
            outs[0].append(y[:b - a])
            outs[1].append(y[b - a:])
        return torch.cat(outs[0] + outs[1]), cache

    whole, c0 = run([0, n])
    for cuts in ([0, 20, 21, n], list(range(n + 1))):
        y, c = run(cuts)
        assert torch.equal(c.k, c0.k) and torch.equal(c.v, c0.v)
        # each path's attention is within 3 roundings of 2^-11 (weight, value, output) of the exact one on values
        # up to max|v|; Q8_1 of the output product re-quantises it in steps of max / 127
        w = wo(torch.eye(heads * dim, device="cuda", dtype=torch.float16)).abs().sum(0).max()
        vmax = ops.kv_read(c, table, torch.tensor([0, n, 2 * n], dtype=torch.int32, device="cuda"), 2 * n)[1].abs().max()
        assert (y - whole).abs().max() <= w * vmax * (6 * 2.0 ** -11 + 1.0 / 127)
    assert mmvq.take_device_status() == 0


def test_refusals_on_the_gpu():
    batch = ref.Batch("F16", 64, 2, 16, [2], [20])
    table, start, kv_len = batch.on_gpu()
    cache = batch.cache(ops)
    q = make_q(batch, 4, "f16")
    for bad in (q.float(), q.bfloat16(), q[:, :3], q[..., :32], q.cpu(), q.clone().requires_grad_()):
        with pytest.raises(AnvilError):
            ops.paged_attention(bad, cache, table, start, kv_len)
    for args in ((table.long(), start, kv_len), (table, start.long(), kv_len), (table, start, kv_len.long()),
                 (table.cpu(), start, kv_len), (table, start[:1], kv_len), (table, start, kv_len[:0]),
                 (table.repeat(2, 1).t().contiguous().t()[:1], start, kv_len), (table[0], start, kv_len)):
        with pytest.raises(AnvilError):
            ops.paged_attention(q, cache, *args)
    with pytest.raises(AnvilError):
        ops.paged_attention(q, cache, table, start, kv_len, out=torch.empty_like(q).float())
    k = torch.randn(2, 2, 64, device="cuda")
    with pytest.raises(AnvilError):
        ops.kv_write(cache, k, k[:1], table, start, kv_len)
    with pytest.raises(AnvilError):
        ops.kv_write(cache, k, k.half(), table, start, kv_len)
    with pytest.raises(AnvilError):
        ops.kv_read(cache, table, start, 2, dtype=torch.float64)
    with pytest.raises(AnvilError):
        ops.kv_read(cache, table, start, 2, out=(k[:1], k))
    assert mmvq.take_device_status() == 0


# ---- the corners of the two kernels' loads and divisions ---------------------------------------

@pytest.mark.parametrize("kind,dtype", [("F16", "f16"), ("BF16", "bf16"), ("Q8_0", "f16"), ("Q4_0", "bf16")])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 2, 4, 8])
@pytest.mark.parametrize("q_lens", [[1, 3], [2, 45]])
def test_attention_pages_smaller_than_a_load(kind, dtype, dim, page, q_lens):
    batch = ref.Batch(kind, dim, 2, page, q_lens, [77, 130], seed=page, wide=1)
    batch.poison()
    check_attention(batch, 4, dtype)


@pytest.mark.parametrize("q_step,kind,dtype", [(2, "Q4_0", "f16"), (17, "F16", "f16"), (17, "Q8_0", "bf16")])
def test_attention_more_sequences_than_threads(q_step, kind, dtype):
    """The place of a share is found in several passes over the batch."""
    lens = [(37 * i) % 90 for i in range(1100)]
    batch = ref.Batch(kind, 64, 1, 16, [(i * 7) % q_step if n else 0 for i, n in enumerate(lens)], lens, seed=12)
    check_attention(batch, 4, dtype)


@pytest.mark.parametrize("kind,dtype", [("F16", "f16"), ("Q8_0", "f16"), ("BF16", "bf16")])
@pytest.mark.parametrize("q_len", [1, 12])
def test_one_high_score_does_not_drown_thousands_of_low_ones(kind, dtype, q_len):
    """The first key's score is 17 above all others', which are equal, and only the others have values.

    Scores are exact.  A weight is rounded by u_p of itself and, in fp16, by 2^-31 of the largest weight at least;
    exponentials and sums take 2^-18 (16 (n + D) 2^-24), and the output is rounded once.
    """
    n, batch_size, kv_heads, dim = 2000, 48, 8, 64
    batch = ref.Batch(kind, dim, kv_heads, 16, [q_len], [n], seed=13)
    x = torch.zeros(batch.k.shape[0], kv_heads, 16, dim)
    batch.v, batch.vs = ref.quantise(kind, torch.ones_like(x))
    p, o = batch.slots(0, 0)
    x[p, :, o, 0] = 17.0
    batch.k, batch.ks = ref.quantise(kind, x)
    key, one = batch.rows_of("k", 0)[0, 0, 0], batch.rows_of("v", 0)[1, 0, 0]
    batch.set_token("v", 0, 0, 0.0)
    q = torch.zeros(batch_size * q_len, 4 * kv_heads, dim, dtype=ref.NP[dtype], device="cuda")
    q[..., 0] = 1.0
    got = ops.paged_attention(q, batch.cache(ops), batch.table.cuda().expand(batch_size, -1).contiguous(),
                              torch.arange(batch_size + 1, dtype=torch.int32, device="cuda") * q_len,
                              torch.full((batch_size,), n, dtype=torch.int32, device="cuda"), scale=1.0)
    seen = (n - q_len + 1 + torch.arange(q_len).double()).repeat(batch_size)[:, None, None]
    w = (seen - 1) * torch.exp(-key)
    want = one * w / (1 + w)
    u = ref.U[ref.NP[dtype]]
    tol = want * (2 * u + (2.0 ** -11 if batch.ks is not None else 0) + 2.0 ** -18 + 16 * (n + dim) * 2.0 ** -24)
    error = (got.cpu().double() - want).abs()
    assert (error <= tol + seen * 2.0 ** -31 + 2.0 ** -25).all(), (error / want).max()


@pytest.mark.parametrize("q_len", [1, 40])
def test_the_longest_sequence(q_len):
    """2^31 - 4096 tokens, one page named over and over: the attention over that page.

    fp32 sums of some 2^31 / 592 / 4 terms a warp, each addition off by 2^-23 of the sum at most: 2^20 2^-23 would be the
    worst of all, reached only if every addition were cut the same way; a step's 16 to 64 keys are one addition, so
    2^16 2^-23 = 2^-7, beside the roundings of weights, values and output (3 of 2^-11).
    """
    batch = ref.Batch("Q4_0", 64, 1, 1024, [q_len], [1024], seed=14, spare=0)
    cache, q = batch.cache(ops), make_q(batch, 1, "f16")
    table, start, kv_len = batch.on_gpu()
    want = ops.paged_attention(q, cache, table, start, kv_len, causal=False).float()
    longest = 2 ** 31 - 4096
    many = torch.zeros(1, 2 ** 21, dtype=torch.int32, device="cuda")
    bar = (2.0 ** -7 + 4 * 2.0 ** -11) * batch.rows_of("v", 0).abs().max()
    for n, status in ((longest, 0), (2 ** 31 - 1, ops.BAD_PAGE)):
        got = ops.paged_attention(q, cache, many, start, torch.tensor([n], dtype=torch.int32).cuda(), causal=False)
        assert (got.float() - want).abs().max() <= bar
        assert mmvq.take_device_status() == status


@pytest.mark.parametrize("kind,dtype", [("Q8_0", "bf16"), ("F16", "f16")])
@pytest.mark.parametrize("q_lens", [[1, 3], [40, 70]])
def test_pages_beyond_the_fourth_gigabyte(kind, dtype, q_lens):
    batch = ref.Batch(kind, 128, 8, 64, q_lens, [500, 200], seed=15, spare=0)
    pages = batch.k.shape[0]
    small = batch.cache(ops)
    big = ops.PagedKVCache(70000, 64, 8, 128, kind)
    assert big.k.numel() * big.k.element_size() > 2 ** 32 + 2 ** 28
    table, start, kv_len = batch.on_gpu()
    far = torch.where(table < 0, table, table + (70000 - pages))
    new = torch.randn(2, batch.rows, 8, 128, generator=batch.gen).to(ref.NP[dtype]).cuda()
    for name in ("k", "v", "k_scale", "v_scale"):
        if getattr(small, name) is not None:
            getattr(big, name)[70000 - pages:].copy_(getattr(small, name))
    q = make_q(batch, 16, dtype)
    rows = torch.tensor([0, 500, 700], dtype=torch.int32).cuda()
    got = []
    for cache, t in ((small, table), (big, far)):
        ops.kv_write(cache, new[0], new[1], t, start, kv_len)
        got.append((ops.paged_attention(q, cache, t, start, kv_len), *ops.kv_read(cache, t, rows, 700)))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    assert mmvq.take_device_status() == 0


@pytest.mark.parametrize("q_len", [1, 60])
def test_a_table_without_pages(q_len):
    batch = ref.Batch("Q8_0", 128, 1, 16, [q_len, 2], [0, 0], spare=1)
    cache, q = batch.cache(ops), make_q(batch, 4, "bf16")
    table, start, kv_len = batch.on_gpu()
    assert table.shape == (2, 0)
    assert (ops.paged_attention(q, cache, table, start, kv_len) == 0).all()
    assert mmvq.take_device_status() == 0
    assert (ops.paged_attention(q, cache, table, start, kv_len + 5) == 0).all()
    assert mmvq.take_device_status() == ops.BAD_PAGE


def test_the_first_call_of_a_process_may_be_captured():
    """Kernels are loaded and their attributes set while a stream captures."""
    import os
    import subprocess
    import sys

    code = """
import torch
from kernel_anvil import kvcache as ops
table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
for rows in (1, 100):
    q = torch.randn(rows, 8, 128, dtype=torch.float16, device="cuda")
    k = torch.randn(rows, 2, 128, dtype=torch.float16, device="cuda")
    start = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    lens = torch.tensor([600], dtype=torch.int32, device="cuda")
    cache = ops.PagedKVCache(40, 16, 2, 128, "Q8_0")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv_write(cache, k, k, table, start, lens)
        out = ops.paged_attention(q, cache, table, start, lens)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.paged_attention(q, cache, table, start, lens)) and bool(out.any())
"""
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    subprocess.run([sys.executable, "-c", code], check=True, env=env, timeout=240)


@pytest.mark.parametrize("kind,dtype", KIND_TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 256])
def test_attention_of_wide_heads_by_pages(kind, dtype, page):
    check_attention(ref.Batch(kind, 256, 2, page, [70, 3, 150], [333, 90, 150], seed=page), 4, dtype)


@pytest.mark.parametrize("kind,dtype", [("F16", "f16"), ("BF16", "bf16"), ("Q8_0", "bf16"), ("Q4_0", "f16")])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [4, 8, 16, 32, 64, 128])
@pytest.mark.parametrize("q_lens", [[1, 2], [40, 70]])
def test_tokens_of_a_page_that_is_not_there_are_left_out(kind, dtype, dim, page, q_lens):
    """Without a causal mask the result is that of the other pages' tokens."""
    batch = ref.Batch(kind, dim, 2, page, q_lens, [150, 400], seed=page + dim)
    batch.poison()
    q, cache = make_q(batch, 4, dtype), batch.cache(ops)
    table, start, kv_len = batch.on_gpu()
    table[1, 1] = batch.k.shape[0]
    got = ops.paged_attention(q, cache, table, start, kv_len, causal=False).cpu().double()
    assert mmvq.take_device_status() == ops.BAD_PAGE
    batch.table[1, 1:-1] = batch.table[1, 2:].clone()
    batch.kv_lens[1] -= page
    want, tol = ref.attention(batch, q.cpu(), dim ** -0.5, False)
    assert ((got - want).abs() <= tol).all()


# ---- the C entry as a host calls it ------------------------------------------------------------

def c_attention(q, cache, table, start, kv_len, out, work, nbytes, causal=1):
    import ctypes

    from kernel_anvil import _native

    b = ops._batch(cache, table, start, kv_len, q.shape[0])
    lib, ref_b = _native.lib(), ctypes.byref(b)
    need = lib.anvil_paged_attention_workspace(cache._ref, ref_b, q.shape[1])
    status = lib.anvil_paged_attention(cache._ref, ref_b, ops.DTYPES[q.dtype], q.data_ptr(), q.stride(0), q.stride(1),
                                       q.shape[1], cache.head_dim ** -0.5, causal, out.data_ptr(), work, nbytes,
                                       torch.cuda.current_stream().cuda_stream)
    return need, status


@pytest.mark.parametrize("kind,dtype", [("Q8_0", "bf16"), ("F16", "f16")])
@pytest.mark.parametrize("q_lens", [[1, 2, 1], [40, 50, 64]])           # the rows kernel, the tile kernel
def test_a_workspace_that_is_not_needed_is_not_written(kind, dtype, q_lens):
    """Tables of 64 tokens at most need no workspace; a pointer that the host passes all the same stays untouched."""
    batch = ref.Batch(kind, 128, 2, 16, q_lens, [64, 50, 64], seed=40)
    cache, q = batch.cache(ops), make_q(batch, 8, dtype)
    table, start, kv_len = batch.on_gpu()
    assert table.shape[1] * 16 <= 64
    want = ops.paged_attention(q, cache, table, start, kv_len)
    scratch = torch.full((1 << 26,), 0x5A, dtype=torch.uint8, device="cuda")   # notes would lie within it
    for nbytes in (0, 1024):
        out = torch.empty_like(want)
        need, status = c_attention(q, cache, table, start, kv_len, out, scratch.data_ptr() + (1 << 25), nbytes)
        assert (need, status) == (0, 0)
        assert torch.equal(out, want)
        assert bool((scratch == 0x5A).all())


@pytest.mark.parametrize("q_lens", [[1, 2], [40, 50]])
def test_the_workspace_is_as_large_as_asked_for(q_lens):
    """Exactly the bytes that the query names are written, none before or behind them."""
    batch = ref.Batch("Q8_0", 128, 2, 16, q_lens, [700, 450], seed=41)
    cache, q = batch.cache(ops), make_q(batch, 8, "bf16")
    table, start, kv_len = batch.on_gpu()
    want = ops.paged_attention(q, cache, table, start, kv_len)
    need, _ = c_attention(q, cache, table, start, kv_len, torch.empty_like(want), None, 0)
    assert need > 0
    scratch = torch.full((need + 8192,), 0x5A, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(want)
    assert c_attention(q, cache, table, start, kv_len, out, scratch.data_ptr() + 4096, need) == (need, 0)
    assert torch.equal(out, want)
    assert bool((scratch[:4096] == 0x5A).all()) and bool((scratch[4096 + need:] == 0x5A).all())


# ---- entries out of range, rows of no sequence -------------------------------------------------

BAD_LENS = [[65, 33], [1000, 33], [2 ** 31 - 1, 33], [-5, 33], [64, -1], [-2 ** 31, 2 ** 31 - 1]]
BAD_STARTS = [[0, 2, 99], [-1, 2, 3], [0, 2 ** 31 - 1, 3], [-2 ** 31, 2, 3]]


@pytest.mark.parametrize("kind,dtype", [("Q8_0", "f32"), ("Q4_0", "bf16"), ("F16", "f16")])
def test_a_write_with_bad_lengths_or_starts_changes_no_other_token(kind, dtype):
    """A sequence with an entry out of range is not written: its cached tokens, and all others, stay bit for bit."""
    batch = ref.Batch(kind, 64, 2, 16, [2, 1], [64, 33], seed=42)
    cache = batch.cache(ops)
    table, start, kv_len = batch.on_gpu()
    assert table.shape[1] * 16 == 64
    new = torch.randn(3, 2, 64, generator=batch.gen).to(ref.NP[dtype]).cuda()
    tensors = [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    before = [t.clone() for t in tensors]
    calls = [(lens, [0, 2, 3]) for lens in BAD_LENS] + [([64, 33], s) for s in BAD_STARTS] + [([70, 130], [0, 2, 99])]
    for lens, starts in calls:
        ops.kv_write(cache, new, new, table, torch.tensor(starts, dtype=torch.int32).cuda(),
                     torch.tensor(lens, dtype=torch.int32).cuda())
        assert mmvq.take_device_status() == ops.BAD_PAGE, (lens, starts)
        for b, n in enumerate(batch.kv_lens):           # the sequences whose entries are all in range are written
            a, z = starts[b], starts[b + 1]
            fine = 0 <= a <= z <= 3 and 0 <= lens[b] <= 64
            p, o = batch.slots(b, torch.arange(n))
            own = torch.arange(n) >= (n - (z - a) if fine else n)
            for t, was in zip(tensors, before):
                got, old = t[p.cuda(), :, o.cuda()].cpu(), was[p.cuda(), :, o.cuda()].cpu()
                assert torch.equal(got[~own], old[~own]), (lens, starts, b)
                assert not own.any() or not torch.equal(got[own], old[own])
        for t, was in zip(tensors, before):
            t.copy_(was)
    ops.kv_write(cache, new, new, table, start, kv_len)
    assert mmvq.take_device_status() == 0


@pytest.mark.parametrize("kind,dtype", [("F16", "f16"), ("BF16", "bf16"), ("Q8_0", "f16"), ("Q4_0", "bf16")])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [4, 8, 16, 32])
@pytest.mark.parametrize("q_lens", [[1, 2], [40, 70]])
def test_a_value_beside_a_page_that_is_not_there_still_counts(kind, dtype, dim, page, q_lens):
    """An infinite value in a tile that every row sees whole but for a missing page; NaN in the masked ones."""
    batch = ref.Batch(kind, dim, 2, page, q_lens, [150, 400], seed=page + dim)
    p, o = batch.slots(1, 3)
    if batch.vs is None:
        batch.v[p, 0, o, 5] = float("inf")
    else:
        batch.vs[p, 0, o, 1] = float("nan")
    q, cache = make_q(batch, 4, dtype), batch.cache(ops)
    table, start, kv_len = batch.on_gpu()
    table[1, 1] = -1
    for causal in (False, True):                 # (the early tile is seen whole in both)
        got = ops.paged_attention(q, cache, table, start, kv_len, causal=causal).cpu()
        assert mmvq.take_device_status() == ops.BAD_PAGE
        rows = got[q_lens[0]:, :2]               # query heads 0 and 1 read key/value head 0
        if batch.vs is None:
            assert (rows[..., 5] == float("inf")).all()
            assert torch.isfinite(rows[..., :5]).all() and torch.isfinite(rows[..., 6:]).all()
        else:
            assert torch.isnan(rows[..., 32:64]).all()
            assert torch.isfinite(rows[..., :32]).all() and torch.isfinite(rows[..., 64:]).all()
        assert torch.isfinite(got[:q_lens[0]]).all() and torch.isfinite(got[:, 2:]).all()


# ---- scales beyond what the products carry -------------------------------------------------------

def set_block(batch, name, b, pos, scale, code):
    """One cached token's scales and codes, all alike."""
    p, o = batch.slots(b, pos)
    codes, scales = (batch.k, batch.ks) if name == "k" else (batch.v, batch.vs)
    scales[p, :, o] = scale
    codes[p, :, o] = code


@pytest.mark.parametrize("kind,scale,code", [("Q8_0", 516.0, 127), ("Q8_0", 6.0e4, 1), ("Q8_0", -512.5, -127),
                                             ("Q8_0", -600.0, 0), ("Q4_0", 8192.0, 0x00), ("Q4_0", -3.0e4, 0x99)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 4), (128, 64), (256, 16)])
@pytest.mark.parametrize("q_lens", [[4, 5, 12], [40, 5, 150]])
def test_a_scale_beyond_the_range_reaches_only_the_rows_that_see_it(kind, scale, code, dim, page, q_lens):
    """A finite scale above 512 (Q8_0) or 8188 (Q4_0) counts as NaN for the rows that see its token, in keys and
    values, and does not reach the others; it reads back as the value that it stands for."""
    kv_lens, at = [70, 30, 400], {0: 68, 1: 27, 2: 395}
    if q_lens[2] == 150:
        at[2] = 300
    for name in "kv":
        batch = ref.Batch(kind, dim, 1, page, q_lens, kv_lens, seed=43)
        clean = ref.Batch(kind, dim, 1, page, q_lens, kv_lens, seed=43)
        for b, pos in at.items():
            set_block(batch, name, b, pos, scale, code)
        q = make_q(batch, 2, "f16")
        cache, (table, start, kv_len) = batch.cache(ops), batch.on_gpu()
        got = ops.paged_attention(q, cache, table, start, kv_len).cpu().double()
        want, tol = ref.attention(clean, q.cpu(), dim ** -0.5, True)
        for b, pos in at.items():
            n, kv, t0 = q_lens[b], kv_lens[b], int(batch.start[b])
            blind = pos - (kv - n)                      # rows 0 .. blind-1 stand before it
            assert 0 < blind < n
            assert ((got - want).abs() <= tol)[t0:t0 + blind].all(), (name, b)
            assert torch.isnan(got[t0 + blind:t0 + n]).all(), (name, b)
        rows = torch.tensor([0, 0, 0, 400], dtype=torch.int32).cuda()
        read = ops.kv_read(cache, table, rows, 400)["kv".index(name)]
        assert torch.equal(read.cpu(), batch.rows_of(name, 2).float())


@pytest.mark.parametrize("kind,scale,codes", [("Q8_0", 512.0, (127, -127)), ("Q4_0", -8188.0, (0x00, 0xFF))])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_lens", [[4, 5], [40, 150]])
def test_the_largest_scales_are_ordinary_ones(kind, scale, codes, dim, q_lens):
    """Values of up to 65504 in some tokens, beside ordinary ones.

    Where some row does not see a tile, 512 is taken as 511.75, 2^-11 of it less: A 2^-11 more than the bound, which has
    A (u_p + u_v) = A 2^-10 in it, so half of the bound more.
    """
    batch = ref.Batch(kind, dim, 1, 16, q_lens, [70, 400], seed=44)
    for i, pos in enumerate((20, 66, 69)):
        set_block(batch, "v", 0, pos, scale, codes[i & 1])
        set_block(batch, "v", 1, pos * 5, scale, codes[i & 1])
    q = make_q(batch, 2, "f16")
    table, start, kv_len = batch.on_gpu()
    for factor in (0.01, 1e-6):
        want, tol = ref.attention(batch, q.cpu(), factor, True)
        got = ops.paged_attention(q, batch.cache(ops), table, start, kv_len, scale=factor).cpu().double()
        assert ((got - want).abs() <= tol * (1.5 if kind == "Q8_0" else 1)).all()
        set_block(batch, "k", 0, 31, scale, codes[0])
        set_block(batch, "k", 1, 31, scale, codes[1])


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 4), (256, 16)])
@pytest.mark.parametrize("q_lens", [[4, 12], [40, 150]])
def test_the_code_that_no_write_makes_stays_with_the_rows_that_see_it(dim, page, q_lens):
    """-128 (outside the type's codes) times the largest scale passes fp16's range."""
    batch, clean = (ref.Batch("Q8_0", dim, 1, page, q_lens, [70, 400], seed=45) for _ in range(2))
    at = {0: 68, 1: 395 if q_lens[1] == 12 else 300}
    for b, pos in at.items():
        set_block(batch, "v", b, pos, 512.0 - 1024.0 * b, -128)
    q = make_q(batch, 2, "f16")
    table, start, kv_len = batch.on_gpu()
    got = ops.paged_attention(q, batch.cache(ops), table, start, kv_len).cpu().double()
    want, tol = ref.attention(clean, q.cpu(), dim ** -0.5, True)
    for b, pos in at.items():
        t0, blind = int(batch.start[b]), pos - (batch.kv_lens[b] - q_lens[b])
        assert ((got - want).abs() <= tol)[t0:t0 + blind].all(), b


def test_starts_and_lengths_out_of_range_are_reported_by_write_and_read():
    batch = ref.Batch("Q8_0", 64, 2, 16, [3, 0, 2], [40, 20, 33], seed=46)
    cache = batch.cache(ops)
    table, start, kv_len = batch.on_gpu()
    new = torch.randn(5, 2, 64, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    write = lambda s, n: ops.kv_write(cache, new, new, table, s, n)  # noqa: E731
    read = lambda s, n: ops.kv_read(cache, table, s, 5)  # noqa: E731
    for call in (write, read):
        call(start, kv_len)
        assert mmvq.take_device_status() == 0
        for s in ([0, 5, 3, 5], [0, 5, 5, 3], [0, 3, 3, 99], [-1, 3, 3, 5], [0, 3, -7, 5], [2 ** 31 - 1, -2 ** 31, 0, 0],
                  [6, 6, 6, 6], [-3, -2, -1, 0]):
            call(i32(s), kv_len)
            assert mmvq.take_device_status() == ops.BAD_PAGE, s
    for lens in ([40, 65, 33], [40, -1, 33], [40, 2 ** 31 - 1, 33]):   # of a sequence without new tokens
        write(start, i32(lens))
        assert mmvq.take_device_status() == ops.BAD_PAGE, lens
    # many sequences, of which one of the last has the bad entry
    many = torch.arange(2001, dtype=torch.int32, device="cuda").clamp(max=5)
    pages, lens = table[:1].expand(2000, -1).contiguous(), torch.full((2000,), 20, dtype=torch.int32, device="cuda")
    for call in (lambda s: ops.kv_write(cache, new, new, pages, s, lens), lambda s: ops.kv_read(cache, pages, s, 5)):
        call(many)
        assert mmvq.take_device_status() == 0
        late = many.clone()
        late[1990] = 4
        call(late)
        assert mmvq.take_device_status() == ops.BAD_PAGE


def test_a_read_does_not_look_at_the_lengths():
    import ctypes

    from kernel_anvil import _native

    batch = ref.Batch("Q8_0", 64, 2, 16, [3, 2], [40, 33], seed=51)
    cache, (table, start, kv_len) = batch.cache(ops), batch.on_gpu()
    b = ops._batch(cache, table, start, kv_len - 2 ** 30, 5)
    k, v = torch.empty(2, 5, 2, 64, device="cuda")
    assert _native.lib().anvil_kv_read(cache._ref, ctypes.byref(b), None, 0, k.data_ptr(), v.data_ptr(),
                                       torch.cuda.current_stream().cuda_stream) == 0
    assert mmvq.take_device_status() == 0
    assert torch.equal(v[:3].cpu(), batch.rows_of("v", 0, 3).float())


@pytest.mark.parametrize("kind", ["Q8_0", "Q4_0"])
@pytest.mark.parametrize("q_len", [1, 100])
def test_queries_at_both_ends_of_bf16_meet_a_scale_that_brings_them_back(kind, q_len):
    """A quantised cache's queries are brought into fp16's range whatever their exponent."""
    batch = ref.Batch(kind, 128, 1, 16, [q_len], [300], seed=49)
    check_attention(batch, 4, "bf16", amp=2.0 ** 122, scale=0.09 * 2.0 ** -122)
    check_attention(batch, 4, "bf16", amp=2.0 ** 112, scale=0.09 * 2.0 ** -112)
    check_attention(batch, 4, "bf16", amp=2.0 ** -121, scale=0.09 * 2.0 ** 121)


def leave_garbage(nbytes):
    """Blocks of the allocator that hold NaN, for the next allocations of that size."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    held = [torch.full((nbytes // 2,), float("nan"), dtype=torch.float16, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("kind,dtype", [("Q8_0", "bf16"), ("F16", "f16")])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("q_lens,lead,rest", [([1, 1], 0, 30), ([0, 0], 0, 30), ([40, 90], 0, 200), ([3, 0], 5, 90),
                                              ([50, 90], 7, 0), ([0], 0, 1), ([], 0, 9)])
def test_rows_of_no_sequence_are_zeros_in_new_outputs(kind, dtype, dim, q_lens, lead, rest):
    """A padded step: rows before the first sequence and behind the last one, where the call makes the output; where
    the caller gives it they stay as they were."""
    batch = ref.Batch(kind, dim, 2, 16, q_lens, [n + 20 for n in q_lens], seed=47)
    cache, total = batch.cache(ops), lead + batch.rows + rest
    table, start, kv_len = batch.on_gpu()
    start = start + lead
    q = torch.randn(total, 4, dim, generator=batch.gen).to(ref.NP[dtype]).cuda()
    out = torch.full_like(q, 7.0)
    ops.paged_attention(q, cache, table, start, kv_len, out=out)
    assert (out[:lead] == 7).all() and (out[lead + batch.rows:] == 7).all()
    out[:lead], out[lead + batch.rows:] = 0, 0
    leave_garbage(q.numel() * 2)
    assert torch.equal(ops.paged_attention(q, cache, table, start, kv_len), out)
    into = tuple(torch.full((total, 2, dim), 7.0, dtype=q.dtype, device="cuda") for _ in range(2))
    ops.kv_read(cache, table, start, total, dtype=q.dtype, out=into)
    leave_garbage(total * 2 * dim * 2)
    for got, t in zip(ops.kv_read(cache, table, start, total, dtype=q.dtype), into):
        assert (t[:lead] == 7).all() and (t[lead + batch.rows:] == 7).all()
        t[:lead], t[lead + batch.rows:] = 0, 0
        assert torch.equal(got, t)
    assert mmvq.take_device_status() == 0


def test_a_padded_step_replays_with_more_and_fewer_rows():
    batch = ref.Batch("Q8_0", 128, 2, 16, [2, 3], [300, 40], seed=48)
    cache = batch.cache(ops)
    table, start, kv_len = batch.on_gpu()
    q = torch.randn(64, 8, 128, generator=batch.gen).bfloat16().cuda()
    ops.paged_attention(q, cache, table, start, kv_len)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention(q, cache, table, start, kv_len)
    for s in ([0, 2, 5], [0, 30, 64], [0, 1, 1], [0, 0, 0], [0, 10, 12]):
        start.copy_(torch.tensor(s, dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(out).all() and (out[s[-1]:] == 0).all()
        given = torch.full_like(q, 7.0)
        ops.paged_attention(q, cache, table, start, kv_len, out=given)
        assert torch.equal(out[:s[-1]], given[:s[-1]]) and (given[s[-1]:] == 7).all()


def test_a_read_into_overlapping_buffers_is_refused():
    batch = ref.Batch("Q8_0", 64, 2, 16, [5], [5], seed=50)
    table, start, _ = batch.on_gpu()
    cache, both = batch.cache(ops), torch.zeros(11, 2, 64, device="cuda")
    for out in ((both[:5], both[:5]), (both[:5], both[4:9]), (both[4:9], both[:5])):
        with pytest.raises(AnvilError, match="overlap"):
            ops.kv_read(cache, table, start, 5, out=out)
    ops.kv_read(cache, table, start, 5, out=(both[5:10], both[:5]))
    assert torch.equal(both[5:10].cpu(), batch.rows_of("k", 0).float())
    assert mmvq.take_device_status() == 0


@pytest.mark.parametrize("kind,dtype", [("Q8_0", "bf16"), ("F16", "f16")])
@pytest.mark.parametrize("q_lens", [[1, 4], [60, 250]])
def test_attention_in_place_and_over_parts_of_its_queries(kind, dtype, q_lens):
    batch = ref.Batch(kind, 128, 2, 16, q_lens, [3000, 900], seed=52)
    cache, n = batch.cache(ops), batch.rows
    table, start, kv_len = batch.on_gpu()
    room = torch.zeros(2 * n + 1, 4, 128, dtype=ref.NP[dtype], device="cuda")
    q = make_q(batch, 4, dtype)
    want = ops.paged_attention(q, cache, table, start, kv_len)
    for at in (1, n - 1):
        for a, b in ((0, at), (at, 0)):
            room[a:a + n] = q
            with pytest.raises(AnvilError, match="overlap"):
                ops.paged_attention(room[a:a + n], cache, table, start, kv_len, out=room[b:b + n])
    wide = torch.zeros(n, 8, 128, dtype=q.dtype, device="cuda")
    with pytest.raises(AnvilError, match="overlap"):    # a strided view that starts where out does
        ops.paged_attention(wide[:, :4], cache, table, start, kv_len, out=wide.view(-1)[:n * 512].view(n, 4, 128))
    room[:n] = q
    assert torch.equal(ops.paged_attention(room[:n], cache, table, start, kv_len, out=room[n:2 * n]), want)
    assert torch.equal(ops.paged_attention(room[:n], cache, table, start, kv_len, out=room[:n]), want)
    assert mmvq.take_device_status() == 0
