"""Plain 64-bit forms of the paged key / value cache operators, and random batches
for their tests."""
import math

import torch

D = 128


def plan_ref(cached, new, table, ring, head, tail, block):
    """The step plan, request by request, on Python lists (table: list of lists, ring:
    list; both are changed in place).  Returns seq_lens, cu, slots, positions, head, tail."""
    n = len(ring)
    seq, cu, slots, pos = [], [0], [], []
    give = []
    for b, (c, k) in enumerate(zip(cached, new)):
        old = -(-c // block)
        if k < 0:
            give += table[b][:old]
            seq.append(0)
            cu.append(cu[-1])
            continue
        for i in range(old, -(-(c + k) // block)):
            table[b][i] = ring[head % n]
            head += 1
        for p in range(c, c + k):
            slots.append(table[b][p // block] * block + p % block)
            pos.append(p)
        seq.append(c + k)
        cu.append(cu[-1] + k)
    for blk in give:
        ring[tail % n] = blk
        tail += 1
    return seq, cu, slots, pos, head, tail


def norm_rope_ref(x, w, eps, pos, rope, theta):
    """x [T, H, 128] in float64 -> RMSNorm (w or None) and rotary embedding."""
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    if rope == "none":
        return x
    i = torch.arange(64, dtype=torch.float64, device=x.device)
    ang = pos.double()[:, None, None] * torch.exp(-math.log(theta) * i / 64)
    c, s = torch.cos(ang), torch.sin(ang)
    y = torch.empty_like(x)
    lo, hi = (slice(0, 64), slice(64, 128)) if rope == "neox" else (slice(0, 128, 2), slice(1, 128, 2))
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., lo] * s + x[..., hi] * c
    return y


class Batch:
    """Requests with `new` tokens on top of `cached` ones, over a cache whose unused
    parts (blocks of nobody, the end of a last block) hold NaN."""

    def __init__(self, new, cached, heads, heads_kv, block, dtype, seed=0, extra_rows=3, stride_pad=0, row_pad=0,
                 q_scale=1.0, spare=5, table_pad=2, poison=float("nan")):
        g = torch.Generator().manual_seed(seed)
        self.new, self.cached, self.heads, self.heads_kv, self.block, self.dtype = new, cached, heads, heads_kv, block, dtype
        self.kv = [c + n for c, n in zip(cached, new)]
        self.tokens = sum(new)
        used = [-(-k // block) if k > 0 else 0 for k in self.kv]
        total = sum(used) + spare
        self.n_blocks = total
        order = torch.randperm(total, generator=g)
        per = heads_kv * block * D
        flat = torch.full((2, total, per + stride_pad), poison, dtype=dtype)
        self.k, self.v = (f[:, :per].unflatten(1, (heads_kv, block, D)) for f in flat.cuda())
        width = max(max(used), 1) + table_pad
        table = torch.full((len(new), width), -7, dtype=torch.int32)  # entries behind a request: never used
        self.keys, self.values = [], []
        at = 0
        for b, (k, u) in enumerate(zip(self.kv, used)):
            ids = order[at:at + u]
            at += u
            table[b, :u] = ids.int()
            keys = torch.randn(max(k, 0), heads_kv, D, generator=g).to(dtype)
            vals = torch.randn(max(k, 0), heads_kv, D, generator=g).to(dtype)
            self.keys.append(keys)
            self.values.append(vals)
            for i in range(u):
                part = slice(i * block, min((i + 1) * block, k))
                n = part.stop - part.start
                self.k[ids[i], :, :n] = keys[part].transpose(0, 1).cuda()
                self.v[ids[i], :, :n] = vals[part].transpose(0, 1).cuda()
        self.table = table.cuda()
        self.seq_lens = torch.tensor([max(k, 0) for k in self.kv], dtype=torch.int32).cuda()
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        self.cu = cu
        self.cu_new = torch.tensor(cu, dtype=torch.int32).cuda()
        self.rows = self.tokens + extra_rows
        q = (q_scale * torch.randn(self.rows, heads * D + row_pad, generator=g)).to(dtype)
        self.q_host = q[:, :heads * D].unflatten(1, (heads, D))
        self.q = q.cuda()[:, :heads * D].unflatten(1, (heads, D))
        self.out = torch.full((self.rows, heads * D + row_pad), 7.0, dtype=dtype).cuda()[:, :heads * D].unflatten(1, (heads, D))
        self.max_new = max(max(new), 1)

    def reference(self, causal, scale=None):
        """(out, bound) in float64 on the GPU: |error| the kernel may have at each value.

        u = eps / 2 of the type.  The output is rounded once: u |o|.  Each softmax
        numerator is rounded once to the type for the matrix product: u A, with A =
        sum p |v| / sum p.  A numerator's own relative error: 2^-13 (the coarsest
        exponential in use), plus that of its exponent, a 128-term f32 dot product,
        128 2^-23 scale sum |q k|, twice because numerator and sum move apart.  The f32
        sums over n keys are chains of at most n / 16 + 32 additions of 2^-23 each."""
        scale = D ** -0.5 if scale is None else scale
        u = torch.finfo(self.dtype).eps / 2
        G = self.heads // self.heads_kv
        out = torch.zeros(self.tokens, self.heads, D, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        for b, n in enumerate(self.new):
            kv = max(self.kv[b], 0)
            if n == 0 or kv == 0:
                continue
            r = slice(self.cu[b], self.cu[b] + n)
            q = self.q[r].double().unflatten(1, (self.heads_kv, G)).permute(1, 2, 0, 3)  # [Hkv, G, n, D]
            k = self.keys[b].cuda().double().permute(1, 0, 2)[:, None]
            v = self.values[b].cuda().double().permute(1, 0, 2)[:, None]
            s = q @ k.transpose(2, 3) * scale
            mag = (q.abs() @ k.abs().transpose(2, 3)).amax(-1, keepdim=True) * scale
            if causal:
                pos = torch.arange(n, device="cuda") + (self.kv[b] - n)
                s = s.masked_fill(torch.arange(kv, device="cuda")[None] > pos[:, None], -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)  # a row without keys: all -inf
            o, a = p @ v, p @ v.abs()
            e = u * (o.abs() + a) + a * (2 ** -13 + 2 * mag * 128 * 2 ** -23 + (kv / 16 + 32) * 2 ** -23)
            out[r] = o.permute(2, 0, 1, 3).flatten(1, 2)
            bound[r] = e.permute(2, 0, 1, 3).flatten(1, 2)
        return out, bound + 1e-30

    def check(self, causal=True, scale=None):
        ref, bound = self.reference(causal, scale)
        got = self.out[:self.tokens].double()
        assert torch.isfinite(got).all(), f"{(~torch.isfinite(got)).sum().item()} values not finite"
        off = (got - ref).abs() / bound
        # Values below the type's smallest normal round to a fixed step.
        tiny = (got - ref).abs() <= torch.finfo(self.dtype).tiny
        off = torch.where(tiny, 0, off)
        assert off.numel() == 0 or off.max().item() <= 1.0, f"error {off.max().item():.3f} of its bound at {off.argmax().item()}"
        assert (self.out[self.tokens:] == 7.0).all(), "rows behind the last request were written"


def row_norm_check(q, k, v, got, scale, u, seen=None, lost=None):
    """The largest error of a row's 128 outputs together, as a share of what it may be:
    q [rows, D], k, v [keys, D] and got [rows, D] in float64, seen [rows, keys] (None:
    all).  v has to be of independent normal values.  `lost`: keys that the reference
    leaves out (a planted mistake).

    A bound per value has to add up every key's rounding as if all had one sign.  Their
    sum over a row's channels does not: numerator j is off by a share t_j of its own, which
    depends on q and k alone, so the error sum_j t_j p_j v_j is a normal vector whose
    channels have a variance of at most t^2 sum p^2, and its norm exceeds 1.5 sqrt(128)
    of that once in 10^13 (chi-square of 128 degrees).  t: a half step u of the type, 2^-13
    for the exponential and 2 mag 128 2^-23 for a 128-term f32 score (Batch.reference).
    The f32 sums take n / 16 + 32 steps at most, each off by 2^-22 of a partial sum, itself
    normal and below 8 sqrt(sum p^2).  The sum of the numerators and the output's own
    rounding move the whole row: u + 2^-13 + 2 mag 128 2^-23 + (n / 16 + 32) 2^-24 of it."""
    s = q @ k.T * scale
    mag = ((q.abs() @ k.abs().T).amax(-1, keepdim=True) * scale)
    if seen is not None:
        s = s.masked_fill(~seen, -math.inf)
    if lost is not None:
        s[:, lost] = -math.inf
    p = torch.softmax(s, -1)
    o = p @ v
    n = k.shape[0]
    spread = p.square().sum(-1, keepdim=True).sqrt() * D ** 0.5
    shift = 2 ** -13 + 2 * mag * 128 * 2 ** -23
    steps = n / 16 + 32
    bound = spread * (1.5 * (u + shift) + steps * 2 ** -19) + o.norm(dim=-1, keepdim=True) * (u + shift + steps * 2 ** -24)
    return ((got - o).norm(dim=-1, keepdim=True) / bound).max().item()
