"""GPU tests of the paged key / value cache: the step plan, the store of keys and
values, attention over the cache, and the three run together, against plain forms
in 64 bits."""
import pytest
import torch

import dcpp_b200
import kv_util
from kv_util import Batch, norm_rope_ref, plan_ref

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype).cuda()


# ------------------------------------------------------------------- plan
class Plan:
    """Device buffers of one plan call, and the same on the host."""

    def __init__(self, cached, new, block, n_blocks, max_blocks, max_tokens, seed=0, head0=0, held=None):
        g = torch.Generator().manual_seed(seed)
        self.block, self.n_blocks, self.max_tokens = block, n_blocks, max_tokens
        self.cached, self.new = list(cached), list(new)
        ids = torch.randperm(n_blocks, generator=g).tolist()
        self.table = [[-1] * max_blocks for _ in cached]
        for b, c in enumerate(cached):
            for i in range(-(-max(c, 0) // block)):
                if i < max_blocks and ids:
                    self.table[b][i] = ids.pop()
        self.head = head0
        self.tail = head0 + len(ids)
        self.ring = [-1] * n_blocks
        for i, x in enumerate(ids):
            self.ring[(head0 + i) % n_blocks] = x
        self.d = dict(cached=ints(cached), new=ints(new), free_blocks=ints(self.ring),
                      free_in=ints([self.head, self.tail], torch.int64), free_out=ints([0, 0], torch.int64),
                      block_table=ints(self.table), seq_lens=ints([9] * len(cached)), cu_new=ints([9] * (len(cached) + 1)),
                      slots=ints([9] * max_tokens), positions=ints([9] * max_tokens))

    def run(self, ctx):
        ctx.kv_plan(dcpp_b200.KVCache(n_blocks=self.n_blocks, block_size=self.block), **self.d)

    def check(self):
        seq, cu, slots, pos, head, tail = plan_ref(self.cached, self.new, self.table, self.ring, self.head, self.tail, self.block)
        pad = self.max_tokens - len(slots)
        want = dict(block_table=self.table, free_blocks=self.ring, free_out=[head, tail], seq_lens=seq, cu_new=cu,
                    slots=slots + [-1] * pad, positions=pos + [0] * pad)
        for k, v in want.items():
            assert self.d[k].tolist() == v, k


@pytest.mark.parametrize("cached,new,block,pad", [
    ([0], [1], 16, 0), ([15], [1], 16, 0), ([16], [1], 16, 3), ([0], [0], 16, 2), ([5], [-1], 16, 1),
    ([0, 0, 0], [-1, -1, 0], 32, 4), ([31, 32, 33, 64], [1, 1, 1, 200], 32, 0), ([1000], [5000], 64, 100),
    ([7, 300, 0, 64, 128], [0, -1, 257, 1, -1], 128, 5), ([255, 256], [2, 300], 256, 0)])
def test_plan_matches_reference(ctx, cached, new, block, pad):
    need = sum(-(-(c + max(n, 0)) // block) for c, n in zip(cached, new))
    width = max(-(-(c + max(n, 0)) // block) for c, n in zip(cached, new)) + 1
    p = Plan(cached, new, block, need + 3, width, sum(max(n, 0) for n in new) + pad, head0=need + 1)  # the ring wraps
    p.run(ctx)
    ctx.synchronize()
    p.check()


@pytest.mark.parametrize("batch,hi,seed", [(1, 20000, 0), (33, 700, 1), (1000, 60, 2), (1025, 3, 3), (8192, 4, 4)])
def test_plan_random_batches(ctx, batch, hi, seed):
    g = torch.Generator().manual_seed(seed)
    cached = torch.randint(0, 300, (batch,), generator=g).tolist()
    new = torch.randint(-1, hi, (batch,), generator=g).tolist()
    tokens = sum(max(n, 0) for n in new)
    need = sum(-(-(c + max(n, 0)) // 16) for c, n in zip(cached, new))
    p = Plan(cached, new, 16, need, -(-(300 + hi) // 16), tokens + 129, seed, head0=10 ** 10 + 7)
    p.run(ctx)
    ctx.synchronize()
    p.check()


def test_plan_in_place_and_a_life_of_requests(ctx):
    """Counters and lengths updated in place over 60 steps of growing, finishing and
    returning requests; no block ever belongs to two requests or to one and the ring."""
    g = torch.Generator().manual_seed(3)
    batch, block, n_blocks, width = 17, 16, 400, 40
    p = Plan([0] * batch, [0] * batch, block, n_blocks, width, 600)
    p.d["seq_lens"] = p.d["cached"]
    p.d["free_out"] = p.d["free_in"]
    lens = [0] * batch
    for _ in range(60):
        p.cached = list(lens)
        p.new = [-1 if torch.rand((), generator=g) < 0.1 or n > 500 else int(torch.randint(0, 34, (), generator=g)) for n in lens]
        p.d["new"].copy_(torch.tensor(p.new, dtype=torch.int32))
        p.run(ctx)
        ctx.synchronize()
        seq, cu, slots, pos, p.head, p.tail = plan_ref(p.cached, p.new, p.table, p.ring, p.head, p.tail, block)
        assert p.d["seq_lens"].tolist() == seq and p.d["cu_new"].tolist() == cu
        assert p.d["slots"].tolist()[:len(slots)] == slots and p.d["positions"].tolist()[:len(pos)] == pos
        assert p.d["free_in"].tolist() == [p.head, p.tail]
        owned = [x for row, n in zip(p.d["block_table"].tolist(), seq) for x in row[:-(-n // block)]]
        free = [p.ring[i % n_blocks] for i in range(p.head, p.tail)]
        assert sorted(owned + free) == list(range(n_blocks))
        lens = seq


@pytest.mark.parametrize("what,cached,new,n_blocks,width,rows,status", [
    ("too few blocks", [0, 16], [17, 16], 3, 4, 40, 6), ("too few rows", [0, 0], [5, 5], 4, 4, 9, 6),
    ("table too narrow", [0, 0], [1, 33], 9, 2, 99, 1), ("negative length", [-1, 4], [1, 1], 9, 4, 9, 1),
    ("length past the table", [65, 0], [0, 1], 9, 4, 9, 1)])
def test_plan_refuses_a_step_as_a_whole(ctx, what, cached, new, n_blocks, width, rows, status):
    p = Plan(cached, new, 16, n_blocks, width, rows)
    p.run(ctx)
    with pytest.raises(dcpp_b200.DcppError) as e:
        ctx.synchronize()
    assert e.value.status == status, what
    assert p.d["cu_new"].tolist() == [0] * (len(cached) + 1) and p.d["seq_lens"].tolist() == cached
    assert p.d["slots"].tolist() == [-1] * rows and p.d["positions"].tolist() == [0] * rows
    assert p.d["free_out"].tolist() == [p.head, p.tail]
    assert p.d["block_table"].tolist() == p.table and p.d["free_blocks"].tolist() == p.ring
    ctx.synchronize()  # reported once, the context works on


@pytest.mark.parametrize("free", [[-1, 3], [5, 4], [0, 10]])
def test_plan_refuses_bad_counters(ctx, free):
    p = Plan([0], [1], 16, 9, 2, 1)
    p.d["free_in"].copy_(torch.tensor(free))
    p.run(ctx)
    with pytest.raises(dcpp_b200.DcppError) as e:
        ctx.synchronize()
    assert e.value.status == 1 and p.d["free_out"].tolist() == free and p.d["slots"].tolist() == [-1]


def test_plan_reports_a_bad_block(ctx):
    p = Plan([3, 3], [1, 1], 16, 4, 2, 2)
    p.d["block_table"][0, 0] = 4
    p.run(ctx)
    with pytest.raises(dcpp_b200.DcppError) as e:
        ctx.synchronize()
    assert e.value.status == 1
    assert p.d["slots"].tolist() == [-1, p.table[1][0] * 16 + 3]


# ------------------------------------------------------------------ store
def store_case(ctx, tokens, heads, heads_kv, block, dtype, rope, norm, seed=0, far=0, in_place=False, row_pad=0, stride_pad=0,
               skip=()):
    g = torch.Generator().manual_seed(seed)
    cols = (heads + 2 * heads_kv) * 128
    gain = torch.exp(0.7 * torch.randn(cols, generator=g))
    buf = (torch.randn(tokens, cols + row_pad, generator=g) * torch.cat([gain, torch.ones(row_pad)])).to(dtype).cuda()
    qkv = buf[:, :cols]
    n_blocks = -(-tokens // block) + 2
    slots = torch.randperm(n_blocks * block, generator=g)[:tokens].int()
    for t in skip:
        slots[t] = -1
    pos = (torch.randint(0, 4096, (tokens,), generator=g) + far).int()
    per = heads_kv * block * 128
    flat = torch.full((2, n_blocks, per + stride_pad), 3.0, dtype=dtype).cuda()
    k, v = (f[:, :per].unflatten(1, (heads_kv, block, 128)) for f in flat)
    wq, wk = (1 + 0.3 * torch.randn(128, generator=g) for _ in range(2)) if norm else (None, None)
    theta = 1e6 if rope == "neox" else 2000.0
    x = qkv.double().unflatten(1, (heads + 2 * heads_kv, 128))
    q = qkv[:, :heads * 128] if in_place else torch.full((tokens, heads * 128 + row_pad), 5.0, dtype=dtype).cuda()[:, :heads * 128]
    before = q.clone()
    ctx.kv_store(dcpp_b200.KVCache(k, v), qkv, heads, pos.cuda(), slots.cuda(), q, norm_q=None if wq is None else wq.cuda(),
                 norm_k=None if wk is None else wk.cuda(), eps=1e-6, rope=rope, theta=theta)
    ctx.synchronize()
    live = (slots >= 0).cuda()
    at = slots.long().cuda()[live]
    u = torch.finfo(dtype).eps / 2

    def close(got, ref, pair_of):
        # Rounded once (u); the f32 norm, sine, cosine and rotation are off by a few 2^-24 of the pair.
        lo, hi = (slice(0, 64), slice(64, 128)) if rope == "neox" else (slice(0, 128, 2), slice(1, 128, 2))
        size = torch.empty_like(ref)
        size[..., lo] = size[..., hi] = torch.hypot(ref[..., lo], ref[..., hi])
        bound = u * ref.abs() + 2 ** -19 * size + torch.finfo(dtype).tiny
        off = ((got.double() - ref).abs() / bound)
        assert off.numel() == 0 or off.max().item() <= 1.0, (pair_of, off.max().item())

    xq = norm_rope_ref(x[:, :heads], None if wq is None else wq.cuda(), 1e-6, pos.cuda(), rope, theta)
    xk = norm_rope_ref(x[:, heads:heads + heads_kv], None if wk is None else wk.cuda(), 1e-6, pos.cuda(), rope, theta)
    close(q[live].unflatten(1, (heads, 128)), xq[live], "q")
    close(k[at // block, :, at % block], xk[live], "k")
    assert torch.equal(v[at // block, :, at % block].double(), x[live][:, heads + heads_kv:])
    assert torch.equal(q[~live], before[~live])
    free = torch.ones(n_blocks * block, dtype=torch.bool, device="cuda")
    free[at] = False
    rest = free.nonzero().flatten()
    assert (k[rest // block, :, rest % block] == 3.0).all() and (v[rest // block, :, rest % block] == 3.0).all()
    assert (flat[:, :, per:] == 3.0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rope", ["neox", "normal", "none"])
@pytest.mark.parametrize("tokens,heads,heads_kv,block,norm", [(1, 32, 8, 16, True), (7, 1, 1, 32, True), (130, 28, 4, 64, False),
                                                             (65, 16, 16, 128, True), (33, 64, 2, 256, True)])
def test_store_matches_reference(ctx, dtype, rope, tokens, heads, heads_kv, block, norm):
    store_case(ctx, tokens, heads, heads_kv, block, dtype, rope, norm, seed=tokens)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rope", ["neox", "normal", "none"])
@pytest.mark.parametrize("heads,heads_kv,norm,in_place", [(28, 4, True, False), (5, 1, False, True), (1, 1, True, True), (40, 8, True, True)])
def test_store_many_tokens(ctx, dtype, rope, heads, heads_kv, norm, in_place):
    """Enough tokens that warps walk them by themselves, with rows of whole slices and of
    odd ends, strides of their own, and skipped tokens."""
    for tokens in (1184, 1185, 2500, 7500):
        store_case(ctx, tokens, heads, heads_kv, 16, dtype, rope, norm, seed=heads, in_place=in_place, row_pad=8 if in_place else 0,
                   stride_pad=8, skip=range(3, tokens, 97))


def test_store_many_tokens_with_bad_slots(ctx):
    n = 8000
    k = torch.zeros(500, 2, 16, 128, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    qkv = torch.ones(n, 6 * 128, dtype=BF16, device="cuda")
    q = torch.zeros(n, 2 * 128, dtype=BF16, device="cuda")
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    slots[17], slots[4000] = 8000, 2 ** 31 - 1
    ctx.kv_store(dcpp_b200.KVCache(k, v), qkv, 2, torch.zeros_like(slots), slots, q, rope="none")
    with pytest.raises(dcpp_b200.DcppError) as e:
        ctx.synchronize()
    assert e.value.status == 1
    rows = k.transpose(1, 2).flatten(0, 1).flatten(1)
    good = torch.ones(n, dtype=torch.bool, device="cuda")
    good[[17, 4000]] = False
    assert (rows[good] == 1).all() and (rows[~good] == 0).all() and (q[good] == 1).all() and (q[~good] == 0).all()


def test_store_far_positions(ctx):
    store_case(ctx, 50, 4, 2, 16, F16, "neox", True, far=1 << 30)


def test_store_strides_in_place_and_skipped_rows(ctx):
    store_case(ctx, 40, 8, 2, 16, BF16, "neox", True, in_place=True, row_pad=72, stride_pad=64, skip=(0, 3, 39))
    store_case(ctx, 40, 8, 2, 16, F16, "normal", True, row_pad=8, stride_pad=8, skip=range(40))


def test_store_reports_slots_outside_the_cache(ctx):
    k = torch.zeros(3, 2, 16, 128, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    qkv = torch.ones(3, 6 * 128, dtype=BF16, device="cuda")
    q = torch.zeros(3, 2 * 128, dtype=BF16, device="cuda")
    ctx.kv_store(dcpp_b200.KVCache(k, v), qkv, 2, ints([0, 1, 2]), ints([48, 5, -1]), q, rope="none")
    with pytest.raises(dcpp_b200.DcppError) as e:
        ctx.synchronize()
    assert e.value.status == 1
    assert (q[1] == 1).all() and (q[0] == 0).all() and (q[2] == 0).all()
    assert k.sum().item() == 2 * 128 and (k[0, :, 5] == 1).all()


# -------------------------------------------------------------- attention
def attend(ctx, s, causal=True, scale=None, workspace=None):
    cache = dcpp_b200.KVCache(s.k, s.v)
    if workspace is None:
        n = ctx.kv_attention_workspace(cache, s.heads, s.max_new)
        workspace = torch.full((n,), 255, dtype=torch.uint8, device="cuda")  # NaN: nothing may rely on its content
    ctx.kv_attention(cache, s.q, s.cu_new, s.seq_lens, s.table, s.max_new, workspace, s.out, causal=causal, scale=scale)


def run(ctx, s, causal=True, scale=None):
    attend(ctx, s, causal, scale)
    ctx.synchronize()
    s.check(causal, scale)


HEADS = [(32, 8), (8, 8), (16, 2), (8, 1), (28, 4), (12, 4), (32, 1), (128, 1)]


@pytest.mark.parametrize("heads,heads_kv", HEADS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_single_tokens(ctx, heads, heads_kv, dtype):
    run(ctx, Batch([1] * 8, [0, 1, 15, 62, 63, 64, 200, 1000], heads, heads_kv, 16, dtype, seed=heads))


@pytest.mark.parametrize("block", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_block_sizes(ctx, block, causal):
    run(ctx, Batch([1, 2, 3, 1, 1], [700, 126, 255, 0, block - 1], 8, 2, block, BF16, seed=block), causal)
    run(ctx, Batch([130, 3, 77], [300, 126, 0], 8, 2, block, F16, seed=block), causal)


@pytest.mark.parametrize("heads,heads_kv", HEADS)
@pytest.mark.parametrize("new,cached", [([2, 5, 8, 3], [100, 0, 555, 64]), ([17, 1, 0, 40], [0, 900, 3, 1]),
                                        ([129, 300, 64], [0, 513, 64]), ([1, 257, 1, 128], [2000, 0, 0, 128])])
def test_attention_chunks(ctx, heads, heads_kv, new, cached):
    run(ctx, Batch(new, cached, heads, heads_kv, 16, BF16, seed=len(new)))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new,cached", [([512], [0]), ([511, 1, 300], [1, 0, 3000]), ([1024, 700], [17, 0])])
def test_attention_prompts(ctx, dtype, causal, new, cached):
    run(ctx, Batch(new, cached, 8, 2, 32, dtype, seed=7), causal)


def test_attention_long_cache_few_rows(ctx):
    run(ctx, Batch([1], [70001], 4, 1, 64, BF16, seed=1))
    run(ctx, Batch([3, 1], [33333, 5], 8, 2, 16, F16, seed=2))
    run(ctx, Batch([40], [20011], 8, 1, 128, BF16, seed=3))


def test_attention_no_keys_and_no_rows(ctx):
    """Requests without new tokens, without keys, and (lengths shorter than the new
    tokens) rows at negative positions: rows that attend to nothing are 0."""
    for causal in (True, False):
        run(ctx, Batch([0, 4, 0, 2, 1], [0, -4, 50, 30, -1], 8, 2, 16, BF16), causal)
        run(ctx, Batch([5, 300], [-3, -200], 8, 2, 16, F16), causal)
        run(ctx, Batch([0, 0], [0, 9], 8, 2, 16, BF16), causal)


def test_attention_strided_rows_and_blocks(ctx):
    run(ctx, Batch([1, 1], [40, 500], 8, 2, 16, BF16, row_pad=8, stride_pad=8))
    run(ctx, Batch([200, 33], [40, 500], 8, 2, 16, BF16, row_pad=4 * 128, stride_pad=128))


def test_attention_scale_and_large_scores(ctx):
    """Scores of several hundred: maxima that grow along the keys, numerators that
    underflow, and a scale of one's own."""
    run(ctx, Batch([1, 3, 200], [3000, 500, 100], 8, 2, 16, BF16, q_scale=60.0))
    run(ctx, Batch([1, 3, 200], [3000, 500, 100], 8, 2, 16, F16, q_scale=30.0), True, 0.3)
    run(ctx, Batch([1, 3, 200], [3000, 500, 100], 8, 2, 16, F16), False, 1e-4)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_growing_scores(ctx, new):
    """Keys that line up with the queries more and more: every tile's maximum exceeds
    the running one."""
    s = Batch([new], [1500], 4, 1, 16, BF16, seed=5)
    torch.manual_seed(5)
    u = torch.randn(128)
    u /= u.norm()
    n = s.kv[0]
    k = (torch.linspace(-40, 40, n)[:, None, None] * u + 0.1 * torch.randn(n, 1, 128)).to(BF16)
    s.keys[0] = k
    flat = s.table[0, :-(-n // 16)].long()
    pad = torch.full((flat.numel() * 16 - n, 1, 128), float("nan"), dtype=BF16)
    s.k[flat] = torch.cat([k, pad]).unflatten(0, (-1, 16)).transpose(1, 2).cuda()
    s.q.copy_((20 * u + 0.2 * torch.randn(s.q.shape)).to(BF16))
    run(ctx, s)


def test_attention_offsets_past_32_bits(ctx):
    """Blocks beyond 2^31 elements and 2^32 bytes of a plane."""
    block, heads_kv, n_blocks = 256, 8, 17000
    s = Batch([1, 70], [900, 300], 8, heads_kv, block, BF16, seed=9)
    k = torch.empty(n_blocks, heads_kv, block, 128, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 32
    move = n_blocks - s.n_blocks
    k[move:], v[move:] = s.k, s.v
    s.k, s.v = k, v
    s.table = torch.where(s.table >= 0, s.table + move, s.table)
    run(ctx, s)
    qkv = torch.randn(1, 32 * 128, device="cuda").to(BF16)
    q = torch.empty(1, 16 * 128, dtype=BF16, device="cuda")
    ctx.kv_store(dcpp_b200.KVCache(k, v), qkv, 16, ints([0]), ints([(n_blocks - 1) * block + 255]), q, rope="none")
    ctx.synchronize()
    assert torch.equal(v[-1, :, 255].flatten(), qkv[0, 24 * 128:])


def test_attention_is_repeatable(ctx):
    for new in ([1] * 5, [70, 1, 333]):
        s = Batch(new, [4000, 3, 900, 17, 300][:len(new)], 32, 8, 16, BF16)
        attend(ctx, s)
        first = s.out.clone()
        for _ in range(3):
            attend(ctx, s)
            assert torch.equal(first, s.out)
        ctx.synchronize()


# A table this wide says that requests may be long, whatever their lengths: units are
# cut into parts and joined.
WIDE = 9000


@pytest.mark.parametrize("heads,heads_kv", [(32, 8), (16, 2), (8, 8), (12, 4), (64, 1)])
@pytest.mark.parametrize("new,cached", [([1] * 7, [0, 1, 63, 64, 3000, 127, 128]), ([3, 1, 4], [700, 0, 2000]),
                                        ([40, 1, 16, 0, 33], [1, 2500, 128, 7, 95]), ([260, 5, 130], [100, 640, 1000])])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention_cut_units(ctx, heads, heads_kv, new, cached, dtype):
    run(ctx, Batch(new, cached, heads, heads_kv, 16, dtype, seed=heads, table_pad=WIDE))


@pytest.mark.parametrize("keys", [1, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 320, 383, 384, 385, 512, 513, 1000])
@pytest.mark.parametrize("table_pad", [2, WIDE])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_one_row_tile(ctx, keys, table_pad, causal):
    """Units of up to 128 rows, around every length at which the work of their two sides changes."""
    new = min(keys, 20)
    run(ctx, Batch([new, 1, new], [keys - new, 3, keys - new + 1], 12, 2, 16, BF16, seed=keys, table_pad=table_pad), causal)


@pytest.mark.parametrize("heads,heads_kv", [(8, 1), (16, 2), (32, 8), (12, 4)])
@pytest.mark.parametrize("new,cached", [([4], [700]), ([4, 0, 6], [900, 30, 3]), ([40], [4000]), ([64, 1], [1000, 0]),
                                        ([33, 2, 0, 17], [2000, 1, 0, 128]), ([6] * 7, [0, 1, 127, 128, 129, 1500, 300]), ([3, 20], [-2, 800])])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_few_units(ctx, heads, heads_kv, new, cached, causal):
    """Units shared by the CTAs of a cluster, of every size: some without a key tile for
    every CTA, requests without rows, rows without keys."""
    for block in (16, 256):
        run(ctx, Batch(new, cached, heads, heads_kv, block, F16 if block == 16 else BF16, seed=heads), causal)


@pytest.mark.parametrize("batch,heads,heads_kv", [(150, 4, 4), (700, 2, 1), (40, 16, 2)])
@pytest.mark.parametrize("table_pad", [2, WIDE])
def test_attention_many_short_requests(ctx, batch, heads, heads_kv, table_pad):
    """More units than CTAs, more requests than threads: sides and slots change hands
    from unit to unit, and units of one and of two row tiles follow one another."""
    g = torch.Generator().manual_seed(batch)
    cached = torch.randint(0, 400, (batch,), generator=g).tolist()
    for hi in (1, 90):
        new = torch.randint(0, hi + 1, (batch,), generator=g).tolist()
        run(ctx, Batch(new, cached, heads, heads_kv, 16, BF16, seed=hi, table_pad=table_pad if batch < 700 else min(table_pad, 300)))


@pytest.mark.parametrize("heads,heads_kv", [(8, 2), (20, 1), (64, 1)])
@pytest.mark.parametrize("table_pad", [0, 300])
def test_attention_alternating_row_tiles(ctx, heads, heads_kv, table_pad):
    """Units of one and of two row tiles in turn, a key tile or two each: the side that
    has nothing to do in a unit may still be at work on the one before, and no slot may
    be filled a second time before it has seen the first."""
    half = 128 // (heads // heads_kv)
    for seed in range(6):
        g = torch.Generator().manual_seed(seed)
        new = [half + 1 + i % half if i % 3 == 0 else 1 + i % half for i in range(240)]
        cached = torch.randint(0, (1, 100, 200)[seed % 3], (240,), generator=g).tolist()
        s = Batch(new, cached, heads, heads_kv, 16, BF16, seed=seed, table_pad=table_pad)
        for _ in range(10):
            attend(ctx, s)
        ctx.synchronize()
        s.check()


@pytest.mark.parametrize("new,cached", [([1], [100]), ([1] * 300, [900] * 300), ([1, 1], [9000, 20]), ([20], [400]), ([20], [9000]), ([200], [100])])
@pytest.mark.parametrize("table_pad", [2, WIDE])
def test_attention_nan_stays_in_its_row(ctx, new, cached, table_pad):
    """A query row with a NaN gives a row of NaN, not one of zeros, and no other row changes."""
    s = Batch(new, cached, 8, 2, 16, BF16, table_pad=table_pad if len(new) < 300 else 2)
    attend(ctx, s)
    want = s.out.clone()
    s.q[s.tokens // 2, 3, 77] = float("nan")
    want[s.tokens // 2, 3] = float("nan")
    attend(ctx, s)
    ctx.synchronize()
    assert torch.equal(s.out.isnan(), want.isnan())
    assert torch.equal(s.out.nan_to_num(0.0), want.nan_to_num(0.0))


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,kv", [(1, 70), (20, 150), (150, 200)])
@pytest.mark.parametrize("table_pad", [2, 600])
def test_attention_bad_key_reaches_every_row_that_sees_it(ctx, bad, new, kv, table_pad):
    """A key of NaN, or a score of +inf, at every place in a tile: the rows that attend to
    it are NaN (as softmax makes them), rows before it and other heads do not change."""
    n = 130 if new > 1 else kv
    s = Batch([new] * n, [kv - new] * n, 8, 2, 16, BF16, seed=kv, table_pad=table_pad)
    s.q[:s.tokens, :4, 5] = 1.0  # of head 0's group: 1 x inf, whatever the other channels
    attend(ctx, s)
    want = s.out.clone()
    first = kv - n if kv - n > 0 else 0
    for b in range(n):
        key = (first + b) % kv
        s.k[s.table[b, key // 16].long(), 0, key % 16, 5] = bad
        rows = want[s.cu[b] + max(0, key - (kv - new)):s.cu[b + 1]]
        rows[:, :4] = float("nan")
    attend(ctx, s)
    ctx.synchronize()
    assert torch.equal(s.out.isnan(), want.isnan())
    assert torch.equal(s.out.nan_to_num(0.0), want.nan_to_num(0.0))


def test_attention_reports_bad_lengths_and_blocks(ctx):
    """A request with a bad block or length is reported; the others are computed."""
    for new in ([1, 1, 1], [200, 130, 1]):
        for what in ("block", "length", "rows"):
            s = Batch(new, [300, 300, 300], 8, 2, 16, BF16)
            if what == "block":
                s.table[1, 2] = s.n_blocks
                s.table[1, 3] = -1
            elif what == "length":
                s.seq_lens[1] = s.table.shape[1] * 16 + 1
            else:
                s.max_new -= 1 if new[0] == 200 else 0
                s.cu_new[3] = s.rows + 1 if new[0] == 1 else s.cu_new[3]
            attend(ctx, s)
            with pytest.raises(dcpp_b200.DcppError) as e:
                ctx.synchronize()
            assert e.value.status == 1, what
            ref, bound = s.reference(True)
            fine = [0, 2] if what != "rows" else ([0, 1] if new[0] == 1 else [1, 2])
            for b in fine:
                r = slice(s.cu[b], s.cu[b + 1])
                assert ((s.out[r].double() - ref[r]).abs() <= bound[r]).all(), (what, b)
            assert (s.out[s.tokens:] == 7.0).all()


def test_attention_refuses(ctx):
    s = Batch([2], [30], 8, 2, 16, BF16)
    cache = dcpp_b200.KVCache(s.k, s.v)
    ws = torch.empty(ctx.kv_attention_workspace(cache, 8, 2), dtype=torch.uint8, device="cuda")

    def refused(status, **kw):
        a = dict(cache=cache, q=s.q, cu_new=s.cu_new, seq_lens=s.seq_lens, block_table=s.table, max_new=2, workspace=ws,
                 out=s.out, causal=True, scale=None)
        a.update(kw)
        with pytest.raises(dcpp_b200.DcppError) as e:
            ctx.kv_attention(**a)
        assert e.value.status == status, kw

    refused(1, workspace=ws[:-16])
    refused(1, workspace=ws[8:])
    refused(1, q=s.q.half())
    refused(1, q=s.q[:, :7], out=s.out[:, :7])
    refused(1, out=s.out[:-1])
    refused(1, out=s.q)
    refused(1, max_new=0)
    refused(1, scale=0.0)
    refused(1, scale=float("nan"))
    refused(1, scale=-1.0)
    refused(1, seq_lens=s.seq_lens.long())
    refused(1, block_table=s.table[0])
    refused(1, cu_new=s.cu_new[:1])
    refused(1, q=s.q.cpu())
    refused(1, q=torch.zeros(5, 8, 132, dtype=BF16, device="cuda")[:, :, :128], out=s.out)
    odd = torch.zeros(5, 8 * 128 + 4, dtype=BF16, device="cuda")
    refused(1, q=odd[:, :1024].unflatten(1, (8, 128)), out=s.out)
    refused(1, q=odd.flatten()[4:4 + 5 * 1024].unflatten(0, (5, 8, 128)), out=s.out)
    wide = Batch([2], [30], 129, 1, 16, BF16)
    refused(2, cache=dcpp_b200.KVCache(wide.k, wide.v), q=wide.q, out=wide.out)
    for shape in ((4, 2, 16, 64), (4, 2, 24, 128), (4, 2, 8, 128), (4, 2, 512, 128)):
        k = torch.zeros(shape, dtype=BF16, device="cuda")
        with pytest.raises(dcpp_b200.DcppError) as e:
            ctx.kv_attention_workspace(dcpp_b200.KVCache(k, k.clone()), 8, 1)
        assert e.value.status == 2, shape
    with pytest.raises(dcpp_b200.DcppError):
        dcpp_b200.KVCache(s.k, s.v.half())
    with pytest.raises(dcpp_b200.DcppError):
        dcpp_b200.KVCache(s.k.transpose(1, 2), s.v.transpose(1, 2))
    with pytest.raises(dcpp_b200.DcppError):
        dcpp_b200.KVCache(torch.zeros(4, 2, 16, 128, device="cuda"), torch.zeros(4, 2, 16, 128, device="cuda"))
    ctx.synchronize()
    run(ctx, s)


def test_store_refuses(ctx):
    k = torch.zeros(3, 2, 16, 128, dtype=BF16, device="cuda")
    cache = dcpp_b200.KVCache(k, k.clone())
    qkv = torch.zeros(3, 8 * 128, dtype=BF16, device="cuda")
    base = dict(cache=cache, qkv=qkv, heads=4, positions=ints([0, 1, 2]), slots=ints([0, 1, 2]),
                q=torch.zeros(3, 4 * 128, dtype=BF16, device="cuda"))
    for kw in (dict(heads=3), dict(q=qkv[:, 128:640]), dict(q=base["q"][:2]), dict(rope="spiral"), dict(positions=None),
               dict(theta=0.0), dict(theta=float("inf")), dict(eps=-1.0), dict(qkv=qkv.float()), dict(slots=ints([0, 1])),
               dict(norm_q=torch.ones(64, device="cuda")), dict(norm_k=torch.ones(128, device="cuda").double())):
        with pytest.raises(dcpp_b200.DcppError) as e:
            ctx.kv_store(**{**base, **kw})
        assert e.value.status == 1, kw
    ctx.kv_store(**{**base, "qkv": qkv[:0], "q": base["q"][:0], "positions": ints([]), "slots": ints([])})  # nothing to do
    ctx.synchronize()


def test_plan_refuses(ctx):
    for kw, status in ((dict(block_size=24), 2), (dict(block_size=8), 2), (dict(n_blocks=1 << 28), 2)):
        p = Plan([0], [1], 16, 4, 2, 1)
        c = dcpp_b200.KVCache(**{**dict(n_blocks=4, block_size=16), **kw})
        if "n_blocks" in kw:
            p.d["free_blocks"] = torch.empty(1 << 28, dtype=torch.int32, device="cuda")
        with pytest.raises(dcpp_b200.DcppError) as e:
            ctx.kv_plan(c, **p.d)
        assert e.value.status == status, kw
    p = Plan([0] * 8193, [0] * 8193, 16, 4, 1, 1)
    with pytest.raises(dcpp_b200.DcppError) as e:
        p.run(ctx)
    assert e.value.status == 2
    p = Plan([0, 0], [1, 1], 16, 4, 2, 1)
    for kw in (dict(new=ints([1])), dict(cu_new=ints([0, 0])), dict(positions=ints([])), dict(free_in=ints([0, 4])),
               dict(block_table=ints([[0, 0]])), dict(cached=torch.tensor([0, 0], dtype=torch.int32))):
        with pytest.raises(dcpp_b200.DcppError) as e:
            ctx.kv_plan(dcpp_b200.KVCache(n_blocks=4, block_size=16), **{**p.d, **kw})
        assert e.value.status == 1, kw
    ctx.synchronize()


def test_attention_refuses_tables_of_nearly_2_31_keys(ctx):
    s = Batch([1], [300], 8, 2, 256, BF16)
    for width, fits in ((8388590, True), (8388600, False)):
        table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
        table[:, :2] = s.table[:, :2]
        s.table = table
        if fits:
            run(ctx, s)
            continue
        with pytest.raises(dcpp_b200.DcppError) as e:
            attend(ctx, s)
        assert e.value.status == 2


def test_layouts_that_share_memory_are_refused(ctx):
    """Blocks or rows expanded from one: writing them makes no sense, and reading on by
    the packed size would leave the storage."""
    one = torch.zeros(1, 2, 16, 128, dtype=BF16, device="cuda")
    with pytest.raises(dcpp_b200.DcppError) as e:
        dcpp_b200.KVCache(one.expand(50, -1, -1, -1), one.clone().expand(50, -1, -1, -1))
    assert e.value.status == 1
    k = torch.zeros(3, 2, 16, 128, dtype=BF16, device="cuda")
    cache = dcpp_b200.KVCache(k, k.clone())
    row = torch.zeros(1, 8 * 128, dtype=BF16, device="cuda")
    q = torch.zeros(3, 4 * 128, dtype=BF16, device="cuda")
    for qkv, dst in ((row.expand(3, -1), q), (row.repeat(3, 1), q[:1].expand(3, -1)), (row.flatten(), q)):
        with pytest.raises(dcpp_b200.DcppError) as e:
            ctx.kv_store(cache, qkv, 4, ints([0, 1, 2]), ints([0, 1, 2]), dst)
        assert e.value.status == 1
    ctx.synchronize()


def test_injected_faults_surface(ctx):
    s = Batch([1], [3], 8, 2, 16, BF16)
    for name, call in (("dcpp_kv_attention", lambda: attend(ctx, s)), ("dcpp_kv_plan", lambda: Plan([0], [1], 16, 4, 2, 1).run(ctx))):
        ctx.inject_fault(name)
        with pytest.raises(dcpp_b200.DcppError) as e:
            call()
        assert e.value.status == 9
    run(ctx, s)


# ------------------------------------------------------- the run together
class Server:
    """Requests served step by step: plan, store, attention on one cache, next to a
    dense float64 history of every request."""

    def __init__(self, batch, heads, heads_kv, block, n_blocks, max_tokens, dtype, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.heads, self.heads_kv, self.block, self.dtype, self.rows = heads, heads_kv, block, dtype, max_tokens
        shape = (n_blocks, heads_kv, block, 128)
        self.k = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        self.v = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        self.cache = dcpp_b200.KVCache(self.k, self.v)
        self.width = n_blocks
        self.lens, self.new = ints([0] * batch), ints([0] * batch)
        self.table = torch.full((batch, n_blocks), -1, dtype=torch.int32, device="cuda")
        self.ring = torch.randperm(n_blocks, generator=self.g).int().cuda()
        self.free = ints([0, n_blocks], torch.int64)
        self.cu, self.slots, self.pos = ints([0] * (batch + 1)), ints([0] * max_tokens), ints([0] * max_tokens)
        self.qkv = torch.zeros(max_tokens, (heads + 2 * heads_kv) * 128, dtype=dtype, device="cuda")
        self.q = self.qkv[:, :heads * 128]  # normalised and turned in place
        self.out = torch.zeros(max_tokens, heads, 128, dtype=dtype, device="cuda")
        self.wq, self.wk = ((1 + 0.2 * torch.randn(128, generator=self.g)).cuda() for _ in range(2))
        self.hist = [[] for _ in range(batch)]

    def workspace(self, ctx, max_new):
        self.ws = torch.empty(ctx.kv_attention_workspace(self.cache, self.heads, max_new), dtype=torch.uint8, device="cuda")
        self.max_new = max_new

    def enqueue(self, ctx):
        ctx.kv_plan(self.cache, self.lens, self.new, self.ring, self.free, self.free, self.table, self.lens, self.cu, self.slots,
                    self.pos)
        ctx.kv_store(self.cache, self.qkv, self.heads, self.pos, self.slots, self.q, norm_q=self.wq, norm_k=self.wk)
        ctx.kv_attention(self.cache, self.q.unflatten(1, (self.heads, 128)), self.cu, self.lens, self.table, self.max_new,
                         self.ws, self.out)

    def load(self, new):
        """Inputs of the next step; returns what check needs."""
        self.new.copy_(torch.tensor(new, dtype=torch.int32))
        x = torch.randn(self.rows, self.qkv.shape[1], generator=self.g).to(self.dtype)
        self.qkv.copy_(x)
        return x

    def check(self, new, x):
        at = 0
        u = torch.finfo(self.dtype).eps / 2
        for b, n in enumerate(new):
            if n < 0:
                self.hist[b] = []
                continue
            H, K = self.heads, self.heads_kv
            rows = x[at:at + n].cuda().double().unflatten(1, (H + 2 * K, 128))
            first = len(self.hist[b])
            pos = torch.arange(first, first + n, device="cuda")
            q = norm_rope_ref(rows[:, :H], self.wq, 1e-6, pos, "neox", 1e6)
            k = norm_rope_ref(rows[:, H:H + K], self.wk, 1e-6, pos, "neox", 1e6)
            self.hist[b] += list(zip(k, rows[:, H + K:]))
            if n == 0:
                continue
            kk = torch.stack([h[0] for h in self.hist[b]]).transpose(0, 1)[:, None]  # [Hkv, 1, keys, D]
            vv = torch.stack([h[1] for h in self.hist[b]]).transpose(0, 1)[:, None]
            qq = q.unflatten(1, (K, H // K)).permute(1, 2, 0, 3)
            s = (qq @ kk.transpose(2, 3)) * 128 ** -0.5
            s = s.masked_fill(torch.arange(kk.shape[2], device="cuda")[None] > pos[:, None], -float("inf"))
            p = torch.softmax(s, -1)
            ref, a = p @ vv, p @ vv.abs()
            mag = (qq.abs() @ kk.abs().transpose(2, 3)).amax(-1, keepdim=True) * 128 ** -0.5
            # As kv_util's bound, and q and k rounded once each: a score is off by 2 u of its magnitude.
            bound = u * (ref.abs() + a) + 2 * a * (2 ** -13 + 2 * u * mag + mag * 2 ** -15)
            got = self.out[at:at + n].double().unflatten(1, (K, H // K)).permute(1, 2, 0, 3)
            assert ((got - ref).abs() <= bound).all(), (b, ((got - ref).abs() / bound).max().item())
            at += n
        assert self.lens.tolist() == [len(h) for h in self.hist]


STEPS = [[40, 7, 0], [1, 1, 200], [1, 1, 1], [-1, 30, 1], [33, 1, -1], [0, 1, 65], [1, 1, 1]]


@pytest.mark.parametrize("dtype,heads,heads_kv,block", [(BF16, 8, 2, 16), (F16, 4, 4, 64)])
def test_plan_store_attention_together(ctx, dtype, heads, heads_kv, block):
    s = Server(3, heads, heads_kv, block, 40, 300, dtype)
    s.workspace(ctx, 200)
    for new in STEPS:
        x = s.load(new)
        s.enqueue(ctx)
        ctx.synchronize()
        s.check(new, x)


@pytest.mark.parametrize("max_new", [1, 200])
def test_step_captured_and_replayed(max_new):
    """One graph of a whole step, replayed with other lengths each time."""
    own = dcpp_b200.Context(0)
    stream = torch.cuda.Stream()
    try:
        s = Server(3, 8, 2, 16, 40, 300, BF16)
        s.workspace(own, max_new)
        with torch.cuda.stream(stream):
            own.use_current_stream()
            s.load([0, 0, 0])
            s.enqueue(own)  # an empty step
            own.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                s.enqueue(own)
            for new in [[min(n, max_new) for n in step] for step in STEPS]:
                x = s.load(new)
                graph.replay()
                own.synchronize()
                s.check(new, x)
        stream.synchronize()
        del graph
    finally:
        own.close()


@pytest.mark.parametrize("new,cached", [([1, 1], [9000, 20]), ([200, 3, 90], [100, 4000, 0])])
def test_cut_units_captured_and_replayed(new, cached):
    """The cut form (two kernels) in a graph, replayed after the lengths have changed: as
    a call of its own gives."""
    own = dcpp_b200.Context(0)
    stream = torch.cuda.Stream()
    try:
        s = Batch(new, cached, 16, 4, 16, BF16, table_pad=WIDE)
        ws = torch.empty(own.kv_attention_workspace(dcpp_b200.KVCache(s.k, s.v), 16, s.max_new), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            own.use_current_stream()
            attend(own, s, workspace=ws)
            own.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                attend(own, s, workspace=ws)
            for shorter in (0, 1, 700):
                lens = [max(k - shorter, n) for k, n in zip(s.kv, new)]
                s.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
                s.out.fill_(7.0)
                attend(own, s, workspace=ws)
                want = s.out.clone()
                s.out.fill_(7.0)
                ws.fill_(255)
                graph.replay()
                own.synchronize()
                assert torch.equal(s.out, want)
                assert not torch.equal(s.out[:s.tokens], torch.full_like(s.out[:s.tokens], 7.0))
            s.kv = lens
            s.keys, s.values = ([x[:n] for x, n in zip(v, lens)] for v in (s.keys, s.values))
            s.check()
        stream.synchronize()
        del graph
    finally:
        own.close()


def test_two_streams_with_their_own_workspaces():
    """Two contexts on two streams, each with its own workspace, at the same time."""
    ctxs = [dcpp_b200.Context(0) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    try:
        for new in ([1] * 6, [150, 1, 300, 2, 2, 90]):
            work = [Batch(new, [3000, 5, 800, 64, 0, 1777], 16, 4, 16, BF16, seed=i) for i in range(2)]
            spaces = []
            for c, s in zip(ctxs, work):
                spaces.append(torch.empty(c.kv_attention_workspace(dcpp_b200.KVCache(s.k, s.v), 16, s.max_new),
                                          dtype=torch.uint8, device="cuda"))
            torch.cuda.synchronize()
            for _ in range(5):
                for c, st, s, ws in zip(ctxs, streams, work, spaces):
                    with torch.cuda.stream(st):
                        c.use_current_stream()
                        attend(c, s, workspace=ws)
            for c, s in zip(ctxs, work):
                c.synchronize()
                s.check()
    finally:
        for c in ctxs:
            c.close()


def test_default_stream(ctx):
    """use_current_stream on torch's default stream: ordered with torch's own work."""
    own = dcpp_b200.Context(0)
    try:
        own.use_current_stream()
        s = Batch([1, 90], [500, 0], 8, 2, 16, BF16)
        s.q.mul_(0.5)
        attend(own, s)
        out = s.out.clone()
        torch.cuda.synchronize()
        s.check()
        assert torch.equal(out, s.out)
    finally:
        own.close()
