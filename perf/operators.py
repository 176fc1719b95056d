"""Cases, inputs and plain forms of three groups of operators around the decode cache and the attention layer:

  attend   one new token per sequence attends every cached token of a paged K/V cache (dense_decode_step)
  fork     one cached sequence continues in several slots of a paged cache (NSAPagedDecodeCache.fork)
  reorder  slot b continues the sequence of slot parents[b], as after a beam-search step (NSAPagedDecodeCache.reorder)
  rope     packed projection rows split into q, k, v and gate logits, q and k rotated by positions on several axes
           (ops.qkv_rope_split), and the reverse for the gradients (ops.qkv_rope_pack)

With `own` false everything here is elementary torch; with `own` true run() calls the framework."""
import math

import torch

own = False

PAGE = 64                          # tokens per page of the cache
BLOCK, STRIDE = 32, 16             # compression block and stride of the cache's compressed rows
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
AXES = 3                           # time, height, width


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # the smallest model of the repository's tests, one user, a short chat: latency only
        dict(name="attend_b1_1k_fp32", op="attend", batch=1, ctx=1024, hq=4, hkv=1, dk=64, dv=64, dtype="fp32",
             ragged=False, window=0),
        # one user of a large model at its full context: too few rows to fill the card without splitting the cache
        dict(name="attend_b1_32k", op="attend", batch=1, ctx=32768, hq=64, hkv=4, dk=128, dv=128, dtype="bf16",
             ragged=False, window=0),
        # a serving batch whose sequences have every length from nothing to the longest, 24 query heads on 2
        dict(name="attend_b37_ragged_fp16", op="attend", batch=37, ctx=16001, hq=24, hkv=2, dk=192, dv=128,
             dtype="fp16", ragged=True, window=0),
        # the decode benchmark's batch and context: bandwidth only
        dict(name="attend_b64_32k", op="attend", batch=64, ctx=32768, hq=64, hkv=4, dk=128, dv=128, dtype="bf16",
             ragged=False, window=0),
        # a second answer to a short question: latency only
        dict(name="fork_b2_1k", op="fork", batch=2, ctx=1000, hkv=4, dk=128, dv=128, dtype="bf16"),
        # 63 samples of one long prompt
        dict(name="fork_b64_32k", op="fork", batch=64, ctx=32749, hkv=4, dk=128, dv=128, dtype="bf16"),
        # beams that all change places, at a length that ends with a page
        dict(name="reorder_b16_4k", op="reorder", batch=16, ctx=4096, hkv=4, dk=192, dv=128, dtype="bf16",
             pattern="cycle"),
        # half of the beams end and continue another one
        dict(name="reorder_b64_16k", op="reorder", batch=64, ctx=16411, hkv=4, dk=128, dv=128, dtype="bf16",
             pattern="beams"),
        # one decode step of a small batch
        dict(name="rope_b8", op="rope", tokens=8, hq=64, hkv=4, dk=192, dv=128, dim=64, dtype="bf16",
             interleaved=False, spread="blocks", backward=False),
        # a prompt with images at the long-context benchmark's heads
        dict(name="rope_32k", op="rope", tokens=32768, hq=64, hkv=4, dk=192, dv=128, dim=64, dtype="bf16",
             interleaved=False, spread="blocks", backward=False),
        # its gradients
        dict(name="rope_32k_backward", op="rope", tokens=32768, hq=64, hkv=4, dk=192, dv=128, dim=64, dtype="bf16",
             interleaved=False, spread="blocks", backward=True),
        # an odd number of rows in 32 bits, neighbouring channels paired, every channel of a head rotated
        dict(name="rope_5003_fp32", op="rope", tokens=5003, hq=12, hkv=4, dk=128, dv=128, dim=128, dtype="fp32",
             interleaved=True, spread="turns", backward=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "fork", "reorder", "rope", "rope"])
    dk, dv = rng.choice([(64, 64), (128, 128), (192, 128)])
    hkv = rng.choice([1, 2, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "rope":
        if dtype == "fp32" and dk == 192:
            dk = 128
        interleaved = rng.random() < 0.5
        dim = rng.choice([d for d in (16, 32, 64, 96, 128) if d <= dk])
        hq = hkv * rng.choice([1, 2, 3, 8, 16])
        tokens = _log(rng, 1, 32768)
        while tokens * (hq * dk + hkv * (dk + dv)) * (4 if dtype == "fp32" else 2) > 800_000_000:
            tokens //= 2
        return dict(op=op, tokens=tokens, hq=hq, hkv=hkv, dk=dk, dv=dv, dim=dim, dtype=dtype, interleaved=interleaved,
                    spread=rng.choice(["blocks", "turns"]), backward=rng.random() < 0.5)
    batch, ctx = _log(rng, 1, 64), _log(rng, 1, 32768)
    if dtype == "fp32" and dk == 192:
        dk = 128
    size = 4 if dtype == "fp32" else 2
    while batch * ctx * hkv * (dk + dv) * size > 4_000_000_000:
        batch = (batch + 1) // 2
    if op == "attend":
        group = rng.choice([1, 2, 4, 7, 8, 12, 16, 32, 64])
        return dict(op=op, batch=batch, ctx=ctx, hq=hkv * group, hkv=hkv, dk=dk, dv=dv, dtype=dtype,
                    ragged=rng.random() < 0.6, window=rng.choice([0, 0, 0, 128, 1000]))
    batch = max(2, batch)
    if op == "fork":
        return dict(op=op, batch=batch, ctx=ctx, hkv=hkv, dk=dk, dv=dv, dtype=dtype)
    pattern = rng.choice(["cycle", "beams"])
    if pattern == "cycle":
        ctx = (ctx + PAGE - 1) // PAGE * PAGE
    return dict(op=op, batch=batch, ctx=min(ctx, 16384), hkv=hkv, dk=dk, dv=dv, dtype=dtype, pattern=pattern)


# --------------------------------------------------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype).mul_(0.5)


def _lengths(case, seed):
    """Cached tokens per sequence; a ragged batch holds every length from 0 to the longest, in another order per seed."""
    batch, ctx = case["batch"], case["ctx"]
    if not case["ragged"] or batch == 1:
        return [ctx] * batch
    lens = [ctx * i // (batch - 1) for i in range(batch)]
    order = torch.randperm(batch, generator=torch.Generator().manual_seed(int(seed)))
    return [lens[i] for i in order.tolist()]


def _pages(tokens):
    return (tokens + PAGE - 1) // PAGE


def _prepare_attend(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    lens = _lengths(case, seed)
    need = [_pages(n) for n in lens]
    pages, width = sum(need) + 1, max(_pages(case["ctx"]), 1)
    order = torch.randperm(pages - 1, generator=torch.Generator().manual_seed(int(seed) + 1)).add_(1).tolist()
    table = torch.zeros(case["batch"], width, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    q = torch.randn(case["batch"], case["hq"], case["dk"], generator=gen, device="cuda", dtype=dtype)
    s = dict(case=case, q=q, scale=case["dk"] ** -0.5)
    k = _normal(gen, dtype, pages, PAGE, case["hkv"], case["dk"])
    v = _normal(gen, dtype, pages, case["hkv"], case["dv"], PAGE)
    lens = torch.tensor(lens, dtype=torch.int32)
    if own:
        from nsa_amd.decode import NSAPagedDecodeCache
        cache = NSAPagedDecodeCache(case["batch"], pages - 1, width * PAGE, case["hkv"], case["dk"], case["dv"],
                                    dtype=dtype)
        cache.k_pool.copy_(k)
        cache.v_pool_t.copy_(v)
        cache.block_table.copy_(table)
        cache.ctx_lens.copy_(lens)
        return dict(s, cache=cache)
    return dict(s, k_pool=k, v_pool_t=v, block_table=table.cuda(), ctx_lens=lens.cuda())


def _rows(tokens):
    """Compressed rows of that many tokens."""
    return (tokens - BLOCK) // STRIDE + 1 if tokens >= BLOCK else 0


def _parents(case, seed):
    """Which slot each slot continues."""
    batch = case["batch"]
    order = torch.randperm(batch, generator=torch.Generator().manual_seed(int(seed) + 2)).tolist()
    parents = list(range(batch))
    if case["pattern"] == "cycle":             # every slot takes the place of another one
        for i, b in enumerate(order):
            parents[b] = order[(i + 1) % batch]
    else:                                      # the second half of `order` ends and continues one of the first half
        keep = (batch + 1) // 2
        for i, b in enumerate(order[keep:]):
            parents[b] = order[i]
    return parents


def _prepare_cache(case, seed):
    """A cache whose slot 0 (fork) or every slot (reorder) holds ctx tokens."""
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    batch, ctx, hkv, dk, dv = (case[x] for x in ("batch", "ctx", "hkv", "dk", "dv"))
    filled = 1 if case["op"] == "fork" else batch
    width = _pages(ctx)
    pages = width * filled + batch             # one more per slot for last pages that cannot be shared
    k = _normal(gen, dtype, filled, ctx, hkv, dk)
    v = _normal(gen, dtype, filled, ctx, hkv, dv)
    s = dict(case=case)
    if case["op"] == "fork":
        s["to"] = list(range(1, batch))
    else:
        s["parents"] = _parents(case, seed)
    if own:
        from nsa_amd.decode import NSAPagedDecodeCache
        cache = NSAPagedDecodeCache(batch, pages, ctx, hkv, dk, dv, block=BLOCK, stride=STRIDE, dtype=dtype)
        for b in range(filled):
            cache.fill(k[b], v[b], seq=b)
        return dict(s, cache=cache)
    z = dict(dtype=dtype, device="cuda")
    rows = _rows(ctx)
    cap = max(((width * PAGE - BLOCK) // STRIDE + 1 + 63) // 64 * 64, 64)
    s.update(k_pool=torch.zeros(pages + 1, PAGE, hkv, dk, **z), v_pool_t=torch.zeros(pages + 1, hkv, dv, PAGE, **z),
             ck=torch.zeros(batch, cap, hkv, dk, **z), cvt=torch.zeros(batch, hkv, dv, cap, **z),
             block_table=torch.zeros(batch, width, dtype=torch.int32, device="cuda"),
             ctx_lens=torch.zeros(batch, dtype=torch.int32, device="cuda"))
    for b in range(filled):
        at = slice(1 + b * width, 1 + (b + 1) * width)
        kp = torch.zeros(width * PAGE, hkv, dk, **z)
        vp = torch.zeros(width * PAGE, hkv, dv, **z)
        kp[:ctx], vp[:ctx] = k[b], v[b]
        s["k_pool"][at] = kp.view(width, PAGE, hkv, dk)
        s["v_pool_t"][at] = vp.view(width, PAGE, hkv, dv).permute(0, 2, 3, 1)
        if rows:
            s["ck"][b, :rows] = k[b].float().unfold(0, BLOCK, STRIDE).mean(-1).to(dtype)
            s["cvt"][b, :, :, :rows] = v[b].float().unfold(0, BLOCK, STRIDE).mean(-1).permute(1, 2, 0).to(dtype)
        s["block_table"][b] = torch.arange(at.start, at.stop, dtype=torch.int32)
        s["ctx_lens"][b] = ctx
    if case["op"] == "fork":                   # where the copies of the last page go: the next free pages
        s["fresh"] = list(range(1 + width, width + batch))
    return s


def _offsets(case):
    nq, nk, nv = case["hq"] * case["dk"], case["hkv"] * case["dk"], case["hkv"] * case["dv"]
    return 0, nq, nq + nk, nq + nk + nv


def _row_length(case):
    return (_offsets(case)[3] + 3 * case["hq"] + 7) // 8 * 8


def _pair_axis(case):
    """The axis whose position turns each pair of channels: a quarter of the pairs follow time, the rest height and
    width; in blocks, or taking turns."""
    pairs = case["dim"] // 2
    time = pairs // 4
    height = (pairs - time) // 2
    if case["spread"] == "turns":
        return [i % AXES for i in range(pairs)]
    return [0] * time + [1] * height + [2] * (pairs - time - height)


def _prepare_rope(case, seed):
    gen, dtype = _generator(seed), DTYPES[case["dtype"]]
    n, hq, hkv, dk, dv = (case[x] for x in ("tokens", "hq", "hkv", "dk", "dv"))
    # runs of text and pictures: a picture's tokens share a time and count height and width, text counts all three
    token = torch.arange(n)
    side = 24
    start = int(torch.randint(0, 4096, (1,), generator=torch.Generator().manual_seed(int(seed))))
    in_picture = (token // (side * side)) % 2 == 1
    at = token % (side * side)
    time = start + torch.where(in_picture, token // (side * side) * (side * side), token)
    height = torch.where(in_picture, time + at // side, time)
    width = torch.where(in_picture, time + at % side, time)
    pairs = case["dim"] // 2
    s = dict(case=case, offsets=_offsets(case), ld=_row_length(case),
             positions=torch.stack([time, height, width]).to(device="cuda", dtype=torch.int32),
             pair_axis=_pair_axis(case),
             axis_of=torch.tensor(_pair_axis(case), device="cuda"),
             inv_freq=10000.0 ** -(torch.arange(pairs, dtype=torch.float32, device="cuda") / pairs))
    if case["backward"]:
        s.update(dq=_normal(gen, dtype, n, hq, dk), dk=_normal(gen, dtype, n, hkv, dk),
                 dv=_normal(gen, dtype, n, hkv, dv), dg=_normal(gen, dtype, n, hq, 3))
    else:
        s["packed"] = _normal(gen, dtype, n, s["ld"])
    return s


def prepare(case, seed):
    if case["op"] == "attend":
        return _prepare_attend(case, seed)
    return _prepare_rope(case, seed) if case["op"] == "rope" else _prepare_cache(case, seed)


# ------------------------------------------------------------------------------------------------------------------ run

def _run_attend(s):
    case = s["case"]
    if own:
        from nsa_amd.decode import dense_decode_step
        return dense_decode_step(s["q"], s["cache"], scale=s["scale"], sliding_window=case["window"], return_lse=True)
    q, hkv, dv = s["q"], case["hkv"], case["dv"]
    batch, hq, dk = q.shape
    pages = s["block_table"].long()
    n = pages.shape[1] * PAGE
    k = s["k_pool"][pages].permute(0, 3, 4, 1, 2).float().reshape(batch, hkv, dk, n)
    v = s["v_pool_t"][pages].permute(0, 2, 1, 4, 3).float().reshape(batch, hkv, n, dv)
    scores = torch.matmul(q.float().view(batch, hkv, hq // hkv, dk) * s["scale"], k)
    key, lens = torch.arange(n, device=q.device), s["ctx_lens"].view(-1, 1, 1, 1)
    hidden = key >= lens
    if case["window"]:
        hidden = hidden | (key < lens - case["window"])
    scores = scores.masked_fill(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
    return out.view(batch, hq, dv).to(q.dtype), (top + torch.log(total)).view(batch, hq)


def _cache_tensors(c):
    return c.k_pool, c.v_pool_t, c.block_table, c.ck, c.cvt, c.ctx_lens


def _run_fork(s):
    if own:
        s["cache"].fork(0, s["to"])
        return _cache_tensors(s["cache"])
    case, table, k, v = s["case"], s["block_table"], s["k_pool"], s["v_pool_t"]
    ctx, rows = case["ctx"], _rows(case["ctx"])
    table[1:] = table[:1]
    if ctx % PAGE:
        fresh = torch.tensor(s["fresh"], device="cuda")
        k[fresh] = k[table[0, -1:].long()]
        v[fresh] = v[table[0, -1:].long()]
        table[1:, -1] = fresh.int()
    s["ck"][1:, :rows] = s["ck"][:1, :rows]
    s["cvt"][1:, :, :, :rows] = s["cvt"][:1, :, :, :rows]
    s["ctx_lens"][1:] = ctx
    return k, v, table, s["ck"], s["cvt"], s["ctx_lens"]


def _run_reorder(s):
    if own:
        s["cache"].reorder(s["parents"])
        return _cache_tensors(s["cache"])
    case, table, k, v = s["case"], s["block_table"], s["k_pool"], s["v_pool_t"]
    ctx, rows = case["ctx"], _rows(case["ctx"])
    parents = torch.tensor(s["parents"], device="cuda")
    moved = torch.nonzero(parents != torch.arange(len(s["parents"]), device="cuda")).view(-1)
    source = parents[moved]
    if ctx % PAGE:                             # a slot that ends keeps its own last page, for a copy of its parent's
        last, theirs = table[moved, -1].long(), table[source, -1].long()
        k[last] = k[theirs]
        v[last] = v[theirs]
        table[moved, :-1] = table[source, :-1]
    else:
        table[moved] = table[source]
    s["ck"][moved, :rows] = s["ck"][source, :rows]
    s["cvt"][moved, :, :, :rows] = s["cvt"][source, :, :, :rows]
    s["ctx_lens"][moved] = s["ctx_lens"][source]
    return k, v, table, s["ck"], s["cvt"], s["ctx_lens"]


def _turn(x, cos, sin, case):
    """x [tokens, heads, dk] with the last `dim` channels of every head rotated, in 32 bits."""
    dim = case["dim"]
    still, x = x[..., :x.shape[-1] - dim].float(), x[..., x.shape[-1] - dim:].float()
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    if case["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([still, y], -1)


def _run_rope(s):
    case = s["case"]
    n, hq, hkv, dk, dv, dim = (case[x] for x in ("tokens", "hq", "hkv", "dk", "dv", "dim"))
    at, ld = s["offsets"], s["ld"]
    if own:
        from nsa_amd import ops
        turn = dict(inv_freq=s["inv_freq"], positions=s["positions"], rope_off=dk - dim, rope_dim=dim,
                    interleaved=case["interleaved"], pair_axis=s["pair_axis"])
        if case["backward"]:
            return ops.qkv_rope_pack(s["dq"], s["dk"], s["dv"], s["dg"], ld, at, **turn)
        return ops.qkv_rope_split(s["packed"], hq, hkv, dk, dv, at, **turn)
    # a position times a frequency runs to thousands of turns: the angle is formed in 64 bits
    angle = (s["positions"][s["axis_of"]].double() * s["inv_freq"].double().unsqueeze(1)).t()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if case["backward"]:
        dtype = s["dq"].dtype
        pad = torch.zeros(n, ld - at[3] - 3 * hq, dtype=dtype, device="cuda")
        return torch.cat([_turn(s["dq"], cos, -sin, case).to(dtype).view(n, -1),
                          _turn(s["dk"], cos, -sin, case).to(dtype).view(n, -1),
                          s["dv"].view(n, -1), s["dg"].view(n, -1), pad], 1)
    packed, dtype = s["packed"], s["packed"].dtype
    q = packed[:, :at[1]].view(n, hq, dk)
    k = packed[:, at[1]:at[2]].view(n, hkv, dk)
    return (_turn(q, cos, sin, case).to(dtype), _turn(k, cos, sin, case).to(dtype),
            packed[:, at[2]:at[3]].reshape(n, hkv, dv), packed[:, at[3]:at[3] + 3 * hq].reshape(n, hq, 3))


def run(state):
    op = state["case"]["op"]
    if op == "attend":
        return _run_attend(state)
    if op == "fork":
        return _run_fork(state)
    return _run_reorder(state) if op == "reorder" else _run_rope(state)


# ----------------------------------------------------------------------------------------------------------------- work

def _size(case):
    return 4 if case["dtype"] == "fp32" else 2


def work(case):
    size = _size(case)
    if case["op"] == "attend":
        batch, hq, hkv, dk, dv = (case[x] for x in ("batch", "hq", "hkv", "dk", "dv"))
        lens = _lengths(case, 0)
        if case["window"]:
            lens = [min(n, case["window"]) for n in lens]
        tokens = sum(lens)
        return dict(bytes=tokens * hkv * (dk + dv) * size + batch * hq * ((dk + dv) * size + 4)
                    + sum(_pages(n) for n in lens) * 4 + batch * 4,
                    flops=2 * tokens * hq * (dk + dv))
    if case["op"] in ("fork", "reorder"):
        batch, ctx, hkv, dk, dv = (case[x] for x in ("batch", "ctx", "hkv", "dk", "dv"))
        rows = _rows(ctx) * hkv * (dk + dv) * size + _pages(ctx) * 4 + 4
        last = PAGE * hkv * (dk + dv) * size if ctx % PAGE else 0
        if case["op"] == "fork":
            read, written = 1, batch - 1
        else:
            read = written = batch if case["pattern"] == "cycle" else batch // 2
        return dict(bytes=(read + written) * (rows + last), flops=0)
    n, hq, hkv, dk, dv = (case[x] for x in ("tokens", "hq", "hkv", "dk", "dv"))
    row = hq * dk + hkv * (dk + dv) + 3 * hq
    return dict(bytes=2 * n * row * size + 4 * AXES * n + 2 * case["dim"], flops=3 * n * (hq + hkv) * case["dim"])


# ---------------------------------------------------------------------------------------------------------------- exact

def _exact_attend(case, seed):
    s = _prepare_attend(case, seed)
    if own:
        c = s["cache"]
        s = dict(s, k_pool=c.k_pool, v_pool_t=c.v_pool_t, block_table=c.block_table, ctx_lens=c.ctx_lens)
    batch, hq, hkv, dv = case["batch"], case["hq"], case["hkv"], case["dv"]
    group = hq // hkv
    out = torch.zeros(batch, hq, dv, dtype=torch.float64, device="cuda")
    lse = torch.full((batch, hq), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s["ctx_lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        ids = s["block_table"][b, :_pages(n)].long()
        for h in range(hkv):
            k = s["k_pool"][ids, :, h].reshape(-1, case["dk"])[first:n].double()
            v = s["v_pool_t"][ids, h].transpose(1, 2).reshape(-1, dv)[first:n].double()
            at = slice(h * group, (h + 1) * group)
            scores = s["scale"] * (s["q"][b, at].double() @ k.t())
            lse[b, at] = torch.logsumexp(scores, -1)
            out[b, at] = torch.softmax(scores, -1) @ v
    return out, lse


def _exact_rope(case, seed):
    s = _prepare_rope(case, seed)
    n, hq, hkv, dk, dv, dim = (case[x] for x in ("tokens", "hq", "hkv", "dk", "dv", "dim"))
    at, pairs = s["offsets"], case["dim"] // 2
    first = [dk - dim + (2 * i if case["interleaved"] else i) for i in range(pairs)]
    second = [c + (1 if case["interleaved"] else pairs) for c in first]
    position = s["positions"].double()
    turn = torch.polar(torch.ones(n, pairs, dtype=torch.float64, device="cuda"), torch.stack(
        [position[s["pair_axis"][i]] * float(s["inv_freq"][i]) for i in range(pairs)], 1))
    if case["backward"]:
        turn = turn.conj()

    def turned(x):
        y = x.double()
        for h in range(x.shape[1]):            # one head at a time: complex 128-bit copies of all would be large
            z = torch.complex(y[:, h, first], y[:, h, second]) * turn
            y[:, h, first], y[:, h, second] = z.real, z.imag
        return y

    if case["backward"]:
        out = torch.zeros(n, s["ld"], dtype=torch.float64, device="cuda")
        out[:, :at[1]] = turned(s["dq"]).view(n, -1)
        out[:, at[1]:at[2]] = turned(s["dk"]).view(n, -1)
        out[:, at[2]:at[3]] = s["dv"].view(n, -1)
        out[:, at[3]:at[3] + 3 * hq] = s["dg"].view(n, -1)
        return out
    packed = s["packed"]
    return (turned(packed[:, :at[1]].reshape(n, hq, dk)), turned(packed[:, at[1]:at[2]].reshape(n, hkv, dk)),
            packed[:, at[2]:at[3]].reshape(n, hkv, dv).double(),
            packed[:, at[3]:at[3] + 3 * hq].reshape(n, hq, 3).double())


def exact(case, seed):
    if case["op"] == "attend":
        return _exact_attend(case, seed)
    return _exact_rope(case, seed) if case["op"] == "rope" else None   # moved rows and pages are not computed


