"""GPU tests of the paged attention's numerics at the edges of its types: values that a
mask hides, weights far below the largest one, and long caches row by row."""
import pytest
import torch

import dcpp_b200
from kv_util import Batch

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
WIDE = 9000  # a table this wide makes the attention cut its units into parts


def attend(ctx, s, causal=True):
    cache = dcpp_b200.KVCache(s.k, s.v)
    ws = torch.full((ctx.kv_attention_workspace(cache, s.heads, s.max_new),), 255, dtype=torch.uint8, device="cuda")
    ctx.kv_attention(cache, s.q, s.cu_new, s.seq_lens, s.table, s.max_new, ws, s.out, causal=causal)
    ctx.synchronize()


def put(s, b):
    """Request b's keys and values (s.keys[b], s.values[b]) into its blocks, NaN behind them."""
    n = s.kv[b]
    ids = s.table[b, :-(-n // s.block)].long()
    for src, dst in ((s.keys[b], s.k), (s.values[b], s.v)):
        pad = torch.full((ids.numel() * s.block - n,) + src.shape[1:], float("nan"), dtype=src.dtype)
        dst[ids] = torch.cat([src, pad]).unflatten(0, (-1, s.block)).transpose(1, 2).cuda()


@pytest.mark.parametrize("new,cached,pad", [(4, 60, 2), (20, 0, 2), (20, 300, 2), (20, 300, WIDE), (150, 0, 2), (150, 1000, WIDE)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_hidden_values_of_any_size_have_no_weight(ctx, new, cached, pad, dtype):
    """Values that causal order hides from a row, as large as the type allows: the row
    is what it is without them.  (2^-126 of 3e38 is not small.)"""
    s = Batch([new], [cached], 8, 2, 16, dtype, table_pad=pad)
    attend(ctx, s)
    want = s.out.clone()
    rows = new // 2
    s.values[0][cached + rows:] = torch.finfo(dtype).max
    put(s, 0)
    attend(ctx, s)
    assert torch.equal(s.out[:rows], want[:rows])


@pytest.mark.parametrize("new,pad", [(1, 2), (20, 2), (20, WIDE), (150, 2)])
def test_values_of_vanishing_weight_vanish(ctx, new, pad):
    """Keys 200 below the largest score (e^-200 < 2^-126) with values of 3e38: no trace
    of them."""
    s = Batch([new], [400], 8, 2, 16, BF16, table_pad=pad)
    s.q[..., 0] = 16.0
    s.keys[0][:, :, 0] = 0.0
    s.keys[0][5::9, :, 0] = -160.0  # 16 * 160 * 128^-0.5 = 226 lower
    s.keys[0][:, :, 1:] *= 0.1
    s.values[0][5::9] = 3e38
    put(s, 0)
    attend(ctx, s)
    big = s.out.clone()
    s.values[0][5::9] = 0.0
    put(s, 0)
    attend(ctx, s)
    assert torch.equal(s.out, big)
    s.check()


@pytest.mark.parametrize("new,kv,pad", [(1, 700, 2), (1, 5000, 2), (1, 30000, 2), (4, 30000, WIDE), (20, 700, 2), (20, 3000, 2),
                                        (20, 30000, WIDE), (300, 900, 2), (300, 30000, 2)])
@pytest.mark.parametrize("lower", [15.0, 16.5, 18.0])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_weights_far_below_the_largest(ctx, new, kv, pad, lower, dtype):
    """One key takes nearly all the weight and has the value 0; the others lie `lower`
    below it and share a value of 1, so what is left of their weights is the output.

    The bound is Batch's and f16's fixed step: numerators are kept 2^13 (up to 16 rows of
    a group) or 2^6 times larger, relative to a maximum that is the largest score or below
    it, so each is off by at most 2^-25 2^-13 or 2^-25 2^-6 of the largest weight besides
    its half step.  Outputs of f16 below 2^-14 (700 e^-18 is 2^-16.5) are themselves
    rounded to multiples of 2^-24: half of that."""
    s = Batch([new], [kv - new], 8, 2, 16, dtype, seed=kv, table_pad=pad)
    s.q.mul_(0.1)
    s.q[..., 0] = 16.0
    s.keys[0].mul_(0.05)
    s.keys[0][:, :, 0] = 0.0
    s.keys[0][0, :, 0] = lower / (16 * 128 ** -0.5)
    s.values[0][:] = 1.0
    s.values[0][0] = 0.0
    put(s, 0)
    attend(ctx, s)
    ref, bound = s.reference(True)
    if dtype == F16:
        bound = bound + kv * 2.0 ** (-38 if new * 4 <= 16 else -31) + 2.0 ** -25
    off = ((s.out[:s.tokens].double() - ref).abs() / bound).max().item()
    assert off <= 1.0, off


@pytest.mark.parametrize("new,pad", [(1, 2), (4, WIDE), (20, 2), (20, WIDE), (150, 2)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scores_of_many_millions(ctx, new, pad, dtype):
    """Scores up to 2^23, thousands apart: each row is the value of its largest key.  The
    numerator (2^lift times the rounding of maximum x scale) and the output are rounded once
    each, the f32 division by the sum is off by 2^-23."""
    s = Batch([new], [700], 8, 2, 16, dtype, table_pad=pad)
    s.q.zero_()
    s.q[..., 0] = 8192.0
    g = torch.Generator().manual_seed(new)
    k = (11000.0 - 64 * torch.randperm(s.kv[0], generator=g)[:, None].expand(-1, 2)).to(dtype)  # 8192 * 11000 * 128^-0.5 < 2^23
    s.keys[0].zero_()
    s.keys[0][:, :, 0] = k
    put(s, 0)
    attend(ctx, s)
    best = torch.stack([k[:s.kv[0] - new + i + 1, 0].float().argmax() for i in range(new)])
    size = k[best, 0].float()
    clear = torch.tensor([(k[:s.kv[0] - new + i + 1, 0].float() == size[i]).sum() == 1 for i in range(new)])
    assert clear.sum() > new // 2 or clear.all()
    u = torch.finfo(dtype).eps / 2
    want = s.values[0][best].double().repeat_interleave(4, 1)  # [new, 8, 128]
    got = s.out[:new].double().cpu()
    assert ((got - want).abs() <= (2 * u + u * u + 2 ** -22) * want.abs() + torch.finfo(dtype).tiny)[clear].all()
