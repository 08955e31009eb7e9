"""The paged cache's operators in 64 bits on the CPU (torch), and the batches that the tests build."""
import torch

NP = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step, relative
KV_MAX = 65024.0  # largest magnitude that the quantised kinds store


def quantise(kind, x):
    """(codes as in the cache, scales) of x (..., D), by the kinds' rules in exact arithmetic."""
    if kind in ("F16", "BF16"):
        return x.to(NP[kind.lower()]), None
    w = x.double().clamp(-KV_MAX, KV_MAX).reshape(*x.shape[:-1], -1, 32)
    nan = w.isnan().any(-1)
    w = torch.where(nan[..., None], torch.zeros_like(w), w)
    mag = w.abs()
    M = mag.amax(-1)
    if kind == "Q8_0":
        d = M / 127
        t = torch.where(M[..., None] > 0, 127 * mag / M[..., None].clamp(min=1e-300), 0)
        codes = (torch.floor(t + 0.5) * torch.sign(w)).to(torch.int8).reshape(x.shape)
    else:
        top = w.gather(-1, (mag == M[..., None]).int().argmax(-1, keepdim=True)).squeeze(-1)
        d = top / -8
        n = torch.where(d[..., None] != 0, torch.floor(w / torch.where(d == 0, 1.0, d)[..., None] + 8.5), 8)
        n = n.clamp(0, 15).to(torch.uint8)
        codes = (n[..., :16] | (n[..., 16:] << 4)).reshape(*x.shape[:-1], x.shape[-1] // 2)
    if kind == "Q8_0":
        codes = torch.where(nan.repeat_interleave(32, -1), torch.zeros_like(codes), codes)
    d = d.half()  # from 64 bits: rounded once
    d[nan] = float("nan")
    return codes, d


def values(kind, codes, scales):
    """What rows of the cache stand for, 64 bits."""
    if kind in ("F16", "BF16"):
        return codes.double()
    d = scales.double().repeat_interleave(32, -1)
    if kind == "Q8_0":
        return codes.double() * d
    b = codes.reshape(*codes.shape[:-1], codes.shape[-1] // 16, 16)
    n = torch.cat([b & 15, b >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    return (n.double() - 8) * d


class Batch:
    """A cache with random contents, a shuffled page table and the ragged lengths given."""

    def __init__(self, kind, dim, kv_heads, page, q_lens, kv_lens, seed=0, spare=3, wide=0, amp=1.0):
        g = torch.Generator().manual_seed(seed)
        self.kind, self.dim, self.kv_heads, self.page = kind, dim, kv_heads, page
        self.q_lens, self.kv_lens = list(q_lens), list(kv_lens)
        need = [-(-n // page) for n in kv_lens]
        pages = sum(need) + spare
        x = [amp * torch.randn(pages, kv_heads, page, dim, generator=g) for _ in range(2)]
        (self.k, self.ks), (self.v, self.vs) = quantise(kind, x[0]), quantise(kind, x[1])
        order = torch.randperm(pages, generator=g)
        cols = max(need + [0]) + wide
        self.table = torch.full((len(need), cols), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].int()
            at += n
        self.free = order[at:]
        starts = [0]
        for n in q_lens:
            starts.append(starts[-1] + n)
        self.start = torch.tensor(starts, dtype=torch.int32)
        self.kv_len = torch.tensor(self.kv_lens, dtype=torch.int32)
        self.rows = starts[-1]
        self.gen = g

    def slots(self, b, pos):
        pos = torch.as_tensor(pos)
        return self.table[b, pos // self.page].long(), pos % self.page

    def rows_of(self, name, b, n=None):
        """Cached values of positions 0 .. n-1 of sequence b: (n, kv_heads, dim), 64 bits."""
        n = self.kv_lens[b] if n is None else n
        p, o = self.slots(b, torch.arange(n))
        s = {"k": self.ks, "v": self.vs}[name]
        return values(self.kind, getattr(self, name)[p, :, o], s[p, :, o] if s is not None else None)

    def poison(self, value=float("nan")):
        """Non-finite values in every slot that no sequence has a token in."""
        used = torch.zeros(self.k.shape[0], self.page, dtype=torch.bool)
        for b, n in enumerate(self.kv_lens):
            p, o = self.slots(b, torch.arange(n))
            used[p, o] = True
        dead = ~used[:, None, :, None]
        for t in (self.k, self.v):
            if t.is_floating_point():
                t.masked_fill_(dead, value)
        for t in (self.ks, self.vs):
            if t is not None:
                t.masked_fill_(dead, value)

    def set_token(self, name, b, pos, value):
        """Every value of one cached token (its scale, in a quantised cache)."""
        p, o = self.slots(b, pos)
        t, s = (self.k, self.ks) if name == "k" else (self.v, self.vs)
        if s is None:
            t[p, :, o] = value
        else:
            s[p, :, o] = value
            if t.dtype == torch.int8:
                t[p, :, o] = 1
            else:
                t[p, :, o] = 0x99

    def cache(self, ops):
        d = lambda t: None if t is None else t.cuda()  # noqa: E731
        return ops.PagedKVCache.from_buffers(self.kind, d(self.k), d(self.v), d(self.ks), d(self.vs))

    def on_gpu(self):
        return self.table.cuda(), self.start.cuda(), self.kv_len.cuda()


def attention(batch, q, scale, causal):
    """(out, bound) in 64 bits: the definition's result, and how far a correct kernel may be from it.

    The kernel rounds each weight p_j to its 16-bit type (u_p), a quantised key or value to fp16 (u_v),
    and sums n products in 32 bits, so with the weighted magnitude A = sum p_j |v_j|:
      |error| <= A (u_p + u_v + 2 max_j |ds_j| + slack) + n 2^-25 max|v| + u_out |out|,
      |ds_j| <= |scale| sum |q k_j| (u_v + (D + 2) 2^-24),  slack = 4 (n + D) 2^-24 + 2^-20 (exponentials)
    where n 2^-25 max|v| is what fp16 weights below 2^-14 lose (the largest weight of a row is about 1),
    and the last term is the output's own rounding.
    """
    T, heads, D = q.shape
    group = heads // batch.kv_heads
    out, tol = torch.zeros(T, heads, D, dtype=torch.float64), torch.zeros(T, heads, D, dtype=torch.float64)
    quant = batch.ks is not None
    u_p = U[torch.bfloat16] if batch.kind == "BF16" else U[torch.float16]
    u_v = U[torch.float16] if quant else 0.0
    for b, n in enumerate(batch.q_lens):
        kv, t0 = batch.kv_lens[b], int(batch.start[b])
        if n == 0 or kv == 0:
            continue
        k, v = batch.rows_of("k", b), batch.rows_of("v", b)
        seen = torch.full((n,), kv) if not causal else (torch.arange(n) + kv - n + 1).clamp(0, kv)
        for h in range(heads):
            x = q[t0:t0 + n, h].double()
            kk, vv = k[:, h // group], v[:, h // group]
            hidden = torch.arange(kv)[None, :] >= seen[:, None]
            s = (scale * (x @ kk.T)).masked_fill(hidden, float("-inf"))
            ds = abs(scale) * (x.abs() @ kk.abs().T) * (u_v + (D + 2) * 2.0 ** -24)
            ds = ds.masked_fill(hidden, 0).amax(-1, keepdim=True)
            p = torch.softmax(s, -1)
            p = torch.where(seen[:, None] > 0, p, torch.zeros_like(p))
            o = torch.zeros(n, D, dtype=torch.float64)
            A = torch.zeros(n, D, dtype=torch.float64)
            fine = torch.isfinite(vv).all()
            if fine:
                o, A = p @ vv, p @ vv.abs()
            else:  # a value that a row does not see does not reach it
                for i in range(n):
                    m = int(seen[i])
                    o[i], A[i] = p[i, :m] @ vv[:m], p[i, :m] @ vv[:m].abs()
            slack = 4 * (kv + D) * 2.0 ** -24 + 2.0 ** -20
            big = vv[torch.isfinite(vv)].abs().max() if torch.isfinite(vv).any() else 0.0
            out[t0:t0 + n, h] = o
            tol[t0:t0 + n, h] = A * (u_p + u_v + 2 * ds + slack) + kv * 2.0 ** -25 * big
    return out, tol + U[q.dtype] * out.abs() * (1 + 2.0 ** -6) + 2.0 ** -24
