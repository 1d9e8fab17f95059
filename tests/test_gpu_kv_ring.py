"""What the step plan does with block ids that lie outside the cache: reported, moved on as
they are, and no other request is touched."""
import pytest
import torch

import dcpp_b200

pytestmark = pytest.mark.gpu

N, BLOCK = 8, 16


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).cuda()


def plan(ctx, cached, new, table, ring, free):
    d = dict(cached=ints(cached), new=ints(new), free_blocks=ints(ring), free_in=ints(free, torch.int64),
             free_out=ints([0, 0], torch.int64), block_table=ints(table), seq_lens=ints([9] * len(cached)),
             cu_new=ints([9] * (len(cached) + 1)), slots=ints([9] * 40), positions=ints([9] * 40))
    ctx.kv_plan(dcpp_b200.KVCache(n_blocks=N, block_size=BLOCK), **d)
    return {k: v.tolist() for k, v in d.items()}


def reported(ctx):
    with pytest.raises(dcpp_b200.DcppError) as e:
        ctx.synchronize()
    assert e.value.status == 1
    ctx.synchronize()  # once


@pytest.mark.parametrize("bad", [-1, N, 2 ** 31 - 1])
def test_a_finished_request_with_a_bad_block(ctx, bad):
    out = plan(ctx, [20, 3], [-1, 1], [[5, bad, -1], [2, -1, -1]], [0, 1, 3, 4, 6, -1, -1, -1], [0, 5])
    reported(ctx)
    assert out["free_blocks"] == [0, 1, 3, 4, 6, 5, bad, -1] and out["free_out"] == [0, 7]
    assert out["seq_lens"] == [0, 4] and out["cu_new"] == [0, 0, 1]
    assert out["slots"] == [2 * BLOCK + 3] + [-1] * 39 and out["positions"] == [3] + [0] * 39


@pytest.mark.parametrize("bad", [-1, N, 2 ** 31 - 1])
def test_a_bad_block_in_the_ring(ctx, bad):
    """The second request draws it; the first and the third have their own."""
    out = plan(ctx, [0, 14, 0], [2, 4, 1], [[-1, -1], [5, -1], [-1, -1]], [7, bad, 3, 0, 1, -1, -1, -1], [0, 5])
    reported(ctx)
    assert out["block_table"] == [[7, -1], [5, bad], [3, -1]] and out["free_out"] == [3, 5]
    assert out["seq_lens"] == [2, 18, 1] and out["cu_new"] == [0, 2, 6, 7]
    s = [7 * BLOCK, 7 * BLOCK + 1, 5 * BLOCK + 14, 5 * BLOCK + 15, -1, -1, 3 * BLOCK]
    assert out["slots"] == s + [-1] * 33 and out["positions"] == [0, 1, 14, 15, 16, 17, 0] + [0] * 33


@pytest.mark.parametrize("new", [1, 30])
def test_attention_over_rows_that_share_blocks(ctx, new):
    """Rows of the table that name the same blocks: each request reads what is there."""
    g = torch.Generator().manual_seed(new)
    k, v = (torch.randn(4, 2, BLOCK, 128, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(2 * new, 8, 128, generator=g).bfloat16().cuda()
    q[new:] = q[:new]
    cache = dcpp_b200.KVCache(k, v)
    ws = torch.empty(ctx.kv_attention_workspace(cache, 8, new), dtype=torch.uint8, device="cuda")
    outs = []
    for table in ([[0, 1, 2], [0, 1, 2]], [[0, 1, 2], [0, 1, 3]]):
        out = torch.empty_like(q)
        ctx.kv_attention(cache, q, ints([0, new, 2 * new]), ints([48, 48]), ints(table), new, ws, out, causal=False)
        ctx.synchronize()
        outs.append(out)
    assert torch.equal(outs[0][:new], outs[0][new:])  # the same question to the same keys
    assert torch.equal(outs[1][:new], outs[0][:new]) and not torch.equal(outs[1][new:], outs[0][new:])
