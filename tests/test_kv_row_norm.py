"""Long caches, row by row: the error of a row's outputs together shows a key tile that was
left out, which a bound per value cannot.  The check itself on the CPU, with mistakes
planted in the reference; the kernels on the GPU."""
import pytest
import torch

import dcpp_b200
from kv_util import Batch, row_norm_check

BF16, F16 = torch.bfloat16, torch.float16
SCALE = 128 ** -0.5


def plain(q, k, v, dtype):
    """Attention with f32 scores and the numerators rounded to the type."""
    s = (q.float() @ k.float().T * SCALE)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return ((p.to(dtype).double() @ v) / p.double().sum(-1, keepdim=True)).to(dtype).double()


@pytest.mark.parametrize("keys,dtype", [(5000, BF16), (33333, F16), (70001, BF16)])
def test_a_lost_tile_is_seen(keys, dtype):
    g = torch.Generator().manual_seed(keys)
    q, k, v = (torch.randn(n, 128, generator=g).to(dtype).double() for n in (4, keys, keys))
    u = torch.finfo(dtype).eps / 2
    got = plain(q, k, v, dtype)
    assert row_norm_check(q, k, v, got, SCALE, u) <= 1.0
    for at in (0, keys // 2, keys - 64):
        assert row_norm_check(q, k, v, got, SCALE, u, lost=slice(at, at + 64)) > 1.0, at
    # The same tile twice is as far off as none of it.
    twice = torch.cat([torch.arange(keys), torch.arange(640, 704)])
    assert row_norm_check(q, k, v, plain(q, k[twice], v[twice], dtype), SCALE, u) > 1.0


@pytest.mark.gpu
@pytest.mark.parametrize("new,cached,heads,heads_kv,block,dtype,pad,causal", [
    ([1], [70001], 4, 1, 64, BF16, 2, True), ([3, 1], [33333, 5], 8, 2, 16, F16, 2, True), ([40], [20011], 8, 1, 128, BF16, 2, True),
    ([1], [5000], 8, 2, 16, BF16, 2, True), ([1, 1, 2], [700, 65, 6000], 12, 4, 32, F16, 400, True),
    ([20], [1500], 8, 2, 16, BF16, 2, True), ([20, 33], [9000, 300], 8, 2, 16, F16, 2, False),
    ([200, 5], [9000, 300], 8, 2, 16, BF16, 2, True), ([300], [500], 16, 4, 256, F16, 0, True)])
def test_rows_of_long_caches(ctx, new, cached, heads, heads_kv, block, dtype, pad, causal):
    s = Batch(new, cached, heads, heads_kv, block, dtype, seed=len(new) + heads, table_pad=pad)
    cache = dcpp_b200.KVCache(s.k, s.v)
    ws = torch.full((ctx.kv_attention_workspace(cache, heads, s.max_new),), 255, dtype=torch.uint8, device="cuda")
    ctx.kv_attention(cache, s.q, s.cu_new, s.seq_lens, s.table, s.max_new, ws, s.out, causal=causal)
    ctx.synchronize()
    u = torch.finfo(dtype).eps / 2
    group = heads // heads_kv
    for b, n in enumerate(new):
        kv = s.kv[b]
        seen = None
        if causal:
            seen = torch.arange(kv, device="cuda")[None] <= (kv - n + torch.arange(n, device="cuda"))[:, None]
        for h in range(heads):
            k, v = (x[b][:, h // group].cuda().double() for x in (s.keys, s.values))
            off = row_norm_check(s.q[s.cu[b]:s.cu[b] + n, h].double(), k, v, s.out[s.cu[b]:s.cu[b] + n, h].double(), SCALE, u, seen)
            assert off <= 1.0, (b, h, off)
