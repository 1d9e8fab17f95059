"""Workloads of the paged key / value cache operators: planning a step, storing
a step's keys and values, attention of new tokens over the cache.

A batch of requests shares one cache of fixed-size blocks.  Each step a request
brings `new` tokens on top of the `cached` ones it already has:

  plan       gives every request the blocks its new tokens need (from a ring of
             free blocks; finished requests, new = -1, give theirs back), and the
             step's maps: token offsets, cache slot and position of every token
  store      RMSNorm and rotary embedding of the step's q and k rows, k and v
             rows into their cache slots
  attention  softmax(q k^T * scale) v of each new token over its request's
             cached keys, grouped key / value heads, causal or not

`own` false: elementary torch operations in 32 bits (rotary angles in 64), rounded
once.  `own` true: the library's entry points.  The lengths of a case follow from
the case alone, the values from the seed.
"""
import math
import os
import random
import sys

import torch

own = False

HEAD_DIM = 128
EPS = 1e-6
THETA = 1e6  # the text encoder's rotary base
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ cases
def _case(op, name, batch, new, cached, heads=32, heads_kv=8, block=16, dtype="bf16", causal=True, norm=True,
          rope="neox", released=0, pad=0, fused=False, lens=1):
    return {"name": name, "op": op, "batch": batch, "new_lo": new[0], "new_hi": new[1], "cached_lo": cached[0],
            "cached_hi": cached[1], "heads": heads, "heads_kv": heads_kv, "block": block, "dtype": dtype,
            "causal": causal, "norm": norm, "rope": rope, "released": released, "pad": pad, "fused": fused,
            "lens": lens}


def listed():
    return [
        # One generated token for each of 64 requests: what a serving loop plans every step (latency).
        _case("plan", "plan_decode_64", 64, (1, 1), (1, 2048), lens=11),
        # A full mixed step: chunks, single tokens, idle and finished requests, a fixed row count behind them.
        _case("plan", "plan_mixed_1000", 1000, (0, 61), (0, 4096), released=37, pad=777, lens=12),
        # The rows of the same 64-request step, the text encoder's heads (32 / 8).
        _case("store", "store_decode_64", 64, (1, 1), (1, 2048), lens=13),
        # The text encoder's batch: 4 prompts of 512 tokens.
        _case("store", "store_prompts_4x512", 4, (512, 512), (0, 0), lens=14),
        # Long documents at far positions, f16, an odd number of query heads per key head, rows of padding.
        _case("store", "store_long_f16", 5, (2500, 4000), (60000, 120000), heads=28, heads_kv=4, block=64, dtype="f16",
              pad=129, lens=15),
        # One request, one token, a short prompt: the smallest call, all latency.
        _case("attention", "decode_1x517", 1, (1, 1), (516, 516), lens=16),
        # A serving step: 64 requests of very different lengths, one token each.
        _case("attention", "decode_64_ragged", 64, (1, 1), (100, 8000), lens=17),
        # One request far into a long document: few rows, a long key axis.
        _case("attention", "decode_1x128k", 1, (1, 1), (131070, 131070), block=64, lens=18),
        # Drafted tokens of 16 requests checked at once: 5 rows x 8 heads per key head, f16.
        _case("attention", "verify_16x5_f16", 16, (5, 5), (700, 4000), heads=16, heads_kv=2, block=32, dtype="f16",
              lens=19),
        # The next chunk of a long prompt over what is cached.
        _case("attention", "chunk_512_over_32k", 1, (512, 512), (32203, 32203), lens=20),
        # The text encoder's batch of prompts, ragged, as views into the fused projection rows.
        _case("attention", "prompts_4_ragged", 4, (301, 512), (0, 0), fused=True, lens=21),
        # Whole long prompts: the largest call.
        _case("attention", "prompts_2x8k", 2, (7900, 8192), (0, 0), block=128, lens=22),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "store", "attention", "attention"])
    heads, heads_kv = rng.choice([(32, 8), (16, 2), (16, 16), (8, 1), (28, 4), (12, 4)])
    common = dict(heads=heads, heads_kv=heads_kv, block=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "f16"]),
                  norm=rng.random() < 0.75, rope=rng.choice(["neox", "neox", "normal"]), causal=rng.random() < 0.8,
                  fused=rng.random() < 0.3, pad=rng.choice([0, 0, rng.randint(1, 200)]), lens=rng.randint(1, 10 ** 6))
    if op == "plan":
        batch = _log(rng, 1, 1000)
        hi = _log(rng, 1, max(1, 32000 // batch))
        c = _case("plan", "", batch, (rng.choice([0, 1]), hi), (0, _log(rng, 1, 4096)),
                  released=rng.randint(0, batch // 4), **common)
    elif op == "store":
        batch = _log(rng, 1, 256)
        hi = _log(rng, 1, max(1, 16000 // batch))
        c = _case("store", "", batch, (max(1, hi // 2), hi), (0, _log(rng, 1, 131072)), **common)
    else:
        kind = rng.choice(["decode", "verify", "chunk", "prompts"])
        if kind == "decode":
            batch = _log(rng, 1, 128)
            new, hi = (1, 1), _log(rng, 1, min(131072, 3000000 // heads_kv // batch))
        elif kind == "verify":
            batch = _log(rng, 1, 32)
            new, hi = (1, rng.randint(2, 8)), _log(rng, 16, min(65536, 3000000 // heads_kv // batch))
        elif kind == "chunk":
            batch = _log(rng, 1, 4)
            top = _log(rng, 16, 1024 // batch)
            new, hi = (max(1, top // 2), top), _log(rng, 64, 32000 // batch)
        else:
            batch = _log(rng, 1, 8)
            top = _log(rng, 16, 8192 // batch)
            new, hi = (max(1, top // 2), top), 1
        c = _case("attention", "", batch, new, (hi // 3 if kind != "prompts" else 0, hi if kind != "prompts" else 0),
                  **common)
    del c["name"]
    return c


def _lengths(case):
    """(cached, new) of every request; new = -1: finished."""
    r = random.Random(case["lens"])
    cached = [r.randint(case["cached_lo"], case["cached_hi"]) for _ in range(case["batch"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["batch"])]
    out = set(r.sample(range(case["batch"]), case["released"]))
    return cached, [-1 if i in out else n for i, n in enumerate(new)]


def work(case):
    cached, new = _lengths(case)
    live = [(c, n) for c, n in zip(cached, new) if n >= 0]
    tokens = sum(n for _, n in live)
    heads, heads_kv, block = case["heads"], case["heads_kv"], case["block"]
    row = HEAD_DIM * 2
    if case["op"] == "plan":
        added = sum(-(-(c + n) // block) - -(-c // block) for c, n in live)
        back = sum(-(-c // block) for c, n in zip(cached, new) if n < 0)
        part = sum(1 for c, n in live if n and c % block)
        rows = tokens + case["pad"]
        return {"bytes": 4 * (3 * case["batch"] + case["batch"] + 1 + 2 * rows + 2 * added + 2 * back + part) + 32,
                "flops": 4 * rows}
    if case["op"] == "store":
        return {"bytes": tokens * (2 * (heads + 2 * heads_kv) * row + 8),
                "flops": tokens * (heads + heads_kv) * HEAD_DIM * 7}
    kv = sum(c + n for c, n in live if n)
    pairs = sum(n * c + n * (n + 1) // 2 if case["causal"] else n * (c + n) for c, n in live)
    return {"bytes": 2 * tokens * heads * row + 2 * kv * heads_kv * row + 4 * kv // block,
            "flops": 4 * HEAD_DIM * heads * pairs}


# ----------------------------------------------------------------- inputs
def prepare(case, seed):
    cached, new = _lengths(case)
    dev, dtype, block = "cuda", DTYPES[case["dtype"]], case["block"]
    heads, heads_kv = case["heads"], case["heads_kv"]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    tokens = sum(max(n, 0) for n in new)
    rows = tokens + case["pad"]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s = {"op": case["op"], "block": block, "heads": heads, "heads_kv": heads_kv, "tokens": tokens, "rows": rows,
         "batch": case["batch"], "cached": ints(cached), "new": ints(new), "norm": case["norm"],
         "neox": case["rope"] == "neox", "causal": case["causal"], "max_new": max(max(new), 1),
         "max_kv": max(max(c + max(n, 0) for c, n in zip(cached, new)), 1)}
    old = [-(-c // block) for c in cached]
    full = [-(-(c + max(n, 0)) // block) for c, n in zip(cached, new)]
    width = s["max_blocks"] = max(max(full), max(old), 1) + 3
    held = old if case["op"] == "plan" else full
    total = s["n_blocks"] = sum(full) + 17
    # The blocks of the requests are scattered over the cache, as they are after many steps.
    order = torch.randperm(total, generator=g, device=dev, dtype=torch.int32)
    counts = ints(held).long()
    start = torch.cumsum(counts, 0) - counts
    col = torch.arange(width, device=dev)
    mine = col < counts[:, None]
    s["table"] = torch.where(mine, order[(start[:, None] + col).clamp(max=total - 1)], -1).to(torch.int32).contiguous()
    s["seq_lens"] = ints([c + max(n, 0) for c, n in zip(cached, new)])
    live = s["new"].clamp(min=0)
    s["cu_new"] = torch.cat([live.new_zeros(1), torch.cumsum(live, 0)]).to(torch.int32)
    if case["op"] == "plan":
        # The ring of free blocks, its head somewhere in the middle: the free ones from head up to tail.
        used = sum(old)
        head = int(torch.randint(0, total, (1,), generator=g, device=dev)) + 3 * total
        free = torch.full((total,), -1, dtype=torch.int32, device=dev)
        free[(head + torch.arange(total - used, device=dev)) % total] = order[used:]
        s["free"], s["free_in"] = free, torch.tensor([head, head + total - used], dtype=torch.int64, device=dev)
        s["free_out"] = torch.zeros(2, dtype=torch.int64, device=dev)
        s["slots"], s["positions"] = torch.zeros(rows, dtype=torch.int32, device=dev), torch.zeros(rows, dtype=torch.int32, device=dev)
        return s
    shape = (total, heads_kv, block, HEAD_DIM)
    s["k"] = torch.randn(shape, generator=g, device=dev, dtype=dtype)
    s["v"] = torch.randn(shape, generator=g, device=dev, dtype=dtype)
    width_qkv = (heads + 2 * heads_kv) * HEAD_DIM
    if case["op"] == "store":
        # Projection rows: a spread of scales over the channels, as trained weights give.
        gain = torch.exp(0.5 * torch.randn(width_qkv, generator=g, device=dev))
        s["qkv"] = (torch.randn(rows, width_qkv, generator=g, device=dev) * gain).to(dtype)
        s["norm_q"] = 1 + 0.2 * torch.randn(HEAD_DIM, generator=g, device=dev)
        s["norm_k"] = 1 + 0.2 * torch.randn(HEAD_DIM, generator=g, device=dev)
        t = torch.arange(rows, device=dev)
        b = torch.searchsorted(s["cu_new"][1:].contiguous(), t.to(torch.int32), right=True).clamp(max=case["batch"] - 1)
        pos = s["cached"][b] + (t - s["cu_new"][b])
        inside = t < tokens
        at = s["table"][b, (pos // block).clamp(max=width - 1)].long() * block + pos % block
        s["slots"] = torch.where(inside, at, -1).to(torch.int32)
        s["positions"] = torch.where(inside, pos, 0).to(torch.int32)
        s["q"] = torch.zeros(rows, heads, HEAD_DIM, dtype=dtype, device=dev)
        return s
    # Queries whose scores spread by about 2: some keys stand out, most share the rest.
    q = (2.0 * torch.randn(rows, width_qkv if case["fused"] else heads * HEAD_DIM, generator=g, device=dev)).to(dtype)
    s["q"] = q[:, :heads * HEAD_DIM].unflatten(1, (heads, HEAD_DIM))
    s["out"] = torch.zeros(rows, heads, HEAD_DIM, dtype=dtype, device=dev)
    return s


# ------------------------------------------------------------ plain forms
def _plan_plain(s):
    block, total, width = s["block"], s["n_blocks"], s["max_blocks"]
    dev = s["table"].device
    cached, new, table, free = s["cached"].long(), s["new"].long(), s["table"].long(), s["free"].long()
    gone, live = new < 0, new.clamp(min=0)
    old = (cached + block - 1) // block
    seq = torch.where(gone, 0, cached + live)
    need = torch.where(gone, 0, (seq + block - 1) // block - old)
    back = torch.where(gone, old, 0)
    need_at, back_at = torch.cumsum(need, 0) - need, torch.cumsum(back, 0) - back
    head, tail = s["free_in"][0], s["free_in"][1]
    col = torch.arange(width, device=dev)
    fresh = free[(head + need_at[:, None] + col - old[:, None]) % total]
    grown = torch.where((col >= old[:, None]) & (col < (old + need)[:, None]), fresh, table)
    cu = torch.cat([live.new_zeros(1), torch.cumsum(live, 0)])
    t = torch.arange(s["rows"], device=dev)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=s["batch"] - 1)
    inside = t < cu[-1]
    pos = torch.where(inside, cached[b] + t - cu[b], 0)
    slots = torch.where(inside, grown[b, pos // block] * block + pos % block, -1)
    k = (torch.arange(total, device=dev) - tail) % total
    ends = torch.cumsum(back, 0)
    owner = torch.searchsorted(ends, k, right=True).clamp(max=s["batch"] - 1)
    given = table[owner, (k - back_at[owner]).clamp(0, width - 1)]
    free = torch.where(k < ends[-1], given, free)
    free_out = torch.stack([head + need.sum(), tail + back.sum()])
    i32 = torch.int32
    return {"table": grown.to(i32), "free": free.to(i32), "free_out": free_out, "seq_lens": seq.to(i32),
            "cu_new": cu.to(i32), "slots": slots.to(i32), "positions": pos.to(i32)}


def _store_plain(s):
    heads, heads_kv, n = s["heads"], s["heads_kv"], s["tokens"]
    x = s["qkv"][:n].float().unflatten(1, (heads + 2 * heads_kv, HEAD_DIM))
    q, k, v = x[:, :heads], x[:, heads:heads + heads_kv], x[:, heads + heads_kv:]
    if s["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["norm_q"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + EPS) * s["norm_k"]
    half = HEAD_DIM // 2
    freq = THETA ** (-torch.arange(half, device=x.device, dtype=torch.float64) / half)
    angle = s["positions"][:n].double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turn(y):
        a, b = (y[..., :half], y[..., half:]) if s["neox"] else (y[..., 0::2], y[..., 1::2])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.cat([a, b], -1) if s["neox"] else torch.stack([a, b], -1).flatten(-2)

    dtype = s["qkv"].dtype
    s["q"][:n] = turn(q).to(dtype)
    at = s["slots"][:n].long()
    s["k"][at // s["block"], :, at % s["block"]] = turn(k).to(dtype)
    s["v"][at // s["block"], :, at % s["block"]] = v.to(dtype)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _attention_plain(s):
    heads, heads_kv, block, n = s["heads"], s["heads_kv"], s["block"], s["max_new"]
    dev, batch, group = s["q"].device, s["batch"], heads // heads_kv
    cu, kv = s["cu_new"].long(), s["seq_lens"].long()
    i = torch.arange(n, device=dev)
    q = s["q"][(cu[:-1, None] + i).clamp(max=s["rows"] - 1)].float()  # [B, n, H, D]
    q = q.unflatten(2, (heads_kv, group)).permute(0, 2, 3, 1, 4).reshape(batch, heads_kv, group * n, HEAD_DIM)
    blocks = s["table"][:, :-(-s["max_kv"] // block)].long().clamp(min=0)

    def rows(cache):
        return cache[blocks].float().transpose(1, 2).flatten(2, 3)  # [B, Hkv, keys, D]

    j = torch.arange(blocks.shape[1] * block, device=dev)
    pos = (kv - (cu[1:] - cu[:-1]))[:, None] + i
    seen = (j < kv[:, None, None]).expand(batch, n, -1)
    if s["causal"]:
        seen = seen & (j <= pos[:, :, None])
    scores = (q @ rows(s["k"]).transpose(2, 3)).mul_(HEAD_DIM ** -0.5).unflatten(2, (group, n))
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = scores.flatten(2, 3) @ rows(s["v"])
    out = torch.where(total > 0, out.unflatten(2, (group, n)) / total, 0)
    t = torch.arange(s["tokens"], device=dev)
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    s["out"][:s["tokens"]] = out[b, :, :, t - cu[b]].flatten(1, 2).to(s["out"].dtype)
    return s["out"]


# ------------------------------------------------------------ own kernels
_kept = {}


def _context():
    """The program's one context, on torch's current stream."""
    if "ctx" not in _kept:
        sys.path.insert(0, os.path.join(os.getcwd(), "diffusers-cpp_b200"))
        import dcpp_b200
        _kept["lib"] = dcpp_b200
        _kept["ctx"] = dcpp_b200.Context(0)
        _kept["ctx"].use_current_stream()
        _kept["ws"] = torch.empty(0, dtype=torch.uint8, device="cuda")
    return _kept["ctx"]


def _cache(s):
    """The handle of the state's cache, made once."""
    if "cache" not in s:
        lib = _kept["lib"]
        s["cache"] = (lib.KVCache(n_blocks=s["n_blocks"], block_size=s["block"]) if s["op"] == "plan"
                      else lib.KVCache(s["k"], s["v"]))
    return s["cache"]


def _run_own(s):
    ctx = _context()
    cache = _cache(s)
    if s["op"] == "plan":
        ctx.kv_plan(cache, s["cached"], s["new"], s["free"], s["free_in"], s["free_out"], s["table"], s["seq_lens"],
                    s["cu_new"], s["slots"], s["positions"])
        return {k: s[k] for k in ("table", "free", "free_out", "seq_lens", "cu_new", "slots", "positions")}
    if s["op"] == "store":
        ctx.kv_store(cache, s["qkv"], s["heads"], s["positions"], s["slots"], s["q"],
                     norm_q=s["norm_q"] if s["norm"] else None, norm_k=s["norm_k"] if s["norm"] else None, eps=EPS,
                     rope="neox" if s["neox"] else "normal", theta=THETA)
        return {"q": s["q"], "k": s["k"], "v": s["v"]}
    need = ctx.kv_attention_workspace(cache, s["heads"], s["max_new"])
    if _kept["ws"].numel() < need:
        _kept["ws"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    ctx.kv_attention(cache, s["q"], s["cu_new"], s["seq_lens"], s["table"], s["max_new"], _kept["ws"], s["out"],
                     causal=s["causal"])
    return s["out"]


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plan_plain, "store": _store_plain, "attention": _attention_plain}[state["op"]](state)


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    cached, new = _lengths(case)
    block, heads, heads_kv = case["block"], case["heads"], case["heads_kv"]
    group, f64 = heads // heads_kv, torch.float64
    if case["op"] == "plan":
        return None  # whole numbers: compared with the plain form's
    first = 0
    if case["op"] == "store":
        q, k, v = s["q"].to(f64), s["k"].to(f64), s["v"].to(f64)
        x = s["qkv"].to(f64).reshape(s["rows"], -1, HEAD_DIM)
        m = torch.arange(HEAD_DIM // 2, device=x.device)
        lo, hi = (m, m + HEAD_DIM // 2) if case["rope"] == "neox" else (2 * m, 2 * m + 1)
        for b, n in enumerate(new):
            r = slice(first, first + n)
            turn = torch.polar(torch.ones(n, 1, 1, dtype=f64, device=x.device),
                               torch.arange(cached[b], cached[b] + n, device=x.device, dtype=f64)[:, None, None]
                               / THETA ** (m.to(f64) * 2 / HEAD_DIM))
            done = []
            for rows, w in ((x[r, :heads], s["norm_q"]), (x[r, heads:heads + heads_kv], s["norm_k"])):
                if case["norm"]:
                    rows = rows / (rows.pow(2).sum(-1, keepdim=True) / HEAD_DIM + EPS).sqrt() * w.to(f64)
                z = torch.complex(rows[..., lo], rows[..., hi]) * turn
                y = torch.empty_like(rows)
                y[..., lo], y[..., hi] = z.real, z.imag
                done.append(y)
            q[r] = done[0]
            at = s["slots"][r].long()
            k[at // block, :, at % block] = done[1]
            v[at // block, :, at % block] = x[r, heads + heads_kv:]
            first += n
        return {"q": q, "k": k, "v": v}
    out = torch.zeros(s["rows"], heads, HEAD_DIM, dtype=f64, device="cuda")
    for b, n in enumerate(new):
        keys = cached[b] + n
        blocks = s["table"][b, :-(-keys // block)].long()
        for h in range(heads_kv if n else 0):
            k = s["k"][blocks, h].reshape(-1, HEAD_DIM)[:keys].to(f64)
            v = s["v"][blocks, h].reshape(-1, HEAD_DIM)[:keys].to(f64)
            for i in range(0, n, 1024):
                q = s["q"][first + i:first + min(i + 1024, n), h * group:(h + 1) * group].to(f64)
                e = torch.einsum("ngd,kd->ngk", q, k) / math.sqrt(HEAD_DIM)
                if case["causal"]:
                    row = torch.arange(cached[b] + i, cached[b] + i + q.shape[0], device="cuda")
                    e = e.masked_fill(torch.arange(keys, device="cuda")[None] > row[:, None, None], -math.inf)
                out[first + i:first + i + q.shape[0], h * group:(h + 1) * group] = torch.softmax(e, -1) @ v
        first += n
    return out
