"""GPU tests of dense decode attention (one new token attends every cached token of a contiguous or paged cache) against a
plain float64 softmax over the same cached tokens.

Bound of the error, from the roundings the kernel makes (u = eps / 2 of the tensors' type, f = 2^-24 of fp32):
  scores    a sum of dk products in fp32, times the scale: |ds| <= (dk + 8) f |scale| sum |q k|
  p         off by 2 ds (numerator and denominator) and by 2^-21 (the exponential); the second product takes it as a rounded
            16-bit value and the rounded rest: off by u^2 of itself, or by 2^-25 where a float16 rest has no smaller step
  sums      a wavefront adds a quarter of the visible keys one after another at worst, then joins: (n / 4 + 64) f
  out       rounded once: u |out|
With A = sum p |v| / l and l >= 1 (the largest p is at least 1),
|out - exact| <= u |out| + A (4 ds + 2^-20 + u^2 + 2 (n / 4 + 64) f) + [float16] 2^-25 n max |v|; the same terms without v and
without the 16-bit ones for the log-sum-exp."""
import math
import random

import pytest
import torch

from tests.util import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"
F = 2.0 ** -24


def make_cache(paged, lens, cap, hkv, dk, dv, dtype, seed, garbage=None):
    """A cache whose sequences hold lens[b] random tokens; everything else in it is `garbage` (or random)."""
    from nsa_amd.decode import NSADecodeCache, NSAPagedDecodeCache
    B = len(lens)
    ks = [randn(n, hkv, dk, seed=seed + 2 * b, scale=0.7, dtype=dtype) for b, n in enumerate(lens)]
    vs = [randn(n, hkv, dv, seed=seed + 2 * b + 1, dtype=dtype) for b, n in enumerate(lens)]
    if paged:
        need = [(n + 63) // 64 for n in lens]
        c = NSAPagedDecodeCache(B, sum(need) + 2, cap, hkv, dk, dv, dtype=dtype, device=DEV)
        ids = list(range(1, sum(need) + 3))
        random.Random(seed).shuffle(ids)
        table = torch.zeros(B, c.max_pages, dtype=torch.int32)
        k_pool = torch.full(c.k_pool.shape, garbage if garbage is not None else 0.0).to(dtype)
        v_pool = torch.full(c.v_pool_t.shape, garbage if garbage is not None else 0.0).to(dtype)
        for b, n in enumerate(lens):
            for p in range(need[b]):
                pg = ids.pop()
                table[b, p] = pg
                m = min(64, n - 64 * p)
                k_pool[pg, :m] = ks[b][64 * p:64 * p + m]
                v_pool[pg, :, :, :m] = vs[b][64 * p:64 * p + m].permute(1, 2, 0)
        c.k_pool.copy_(k_pool)
        c.v_pool_t.copy_(v_pool)
        c.block_table.copy_(table)
    else:
        c = NSADecodeCache(B, cap, hkv, dk, dv, dtype=dtype, device=DEV)
        if garbage is not None:
            c.k.fill_(garbage)
            c.vt.fill_(garbage)
        for b, n in enumerate(lens):
            c.k[b, :n] = ks[b].to(DEV)
            c.vt[b, :, :, :n] = vs[b].permute(1, 2, 0).to(DEV)
    c.ctx_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    return c, ks, vs


def plain(q, k, v, scale, window):
    """q [Hq,Dk], k [n,Hkv,Dk], v [n,Hkv,Dv] -> float64 out [Hq,Dv], lse [Hq] and the error bounds of both."""
    hq, hkv, n = q.shape[0], k.shape[1], k.shape[0]
    u, half = torch.finfo(q.dtype).eps / 2, q.dtype == torch.float16
    lo = max(0, n - window) if window else 0
    q, k, v = q.double(), k.double()[lo:], v.double()[lo:]
    if n == 0:
        z = torch.zeros(hq, v.shape[2], dtype=torch.float64, device=q.device)
        return z, torch.full((hq,), -math.inf, dtype=torch.float64, device=q.device), z, z[:, 0]
    qg = q.view(hkv, hq // hkv, -1)
    kt = k.permute(1, 2, 0).contiguous()
    vh = v.transpose(0, 1).contiguous()
    s = scale * torch.matmul(qg, kt)
    p = torch.softmax(s, -1)
    out = torch.matmul(p, vh).reshape(hq, -1)
    A = torch.matmul(p, vh.abs()).reshape(hq, -1)
    lse = torch.logsumexp(s, -1).reshape(hq)
    ds = ((q.shape[1] + 8) * F * abs(scale) * torch.matmul(qg.abs(), kt.abs()).amax(-1)).reshape(hq)
    chain = 2 * ((n - lo) / 4 + 64) * F
    tol = u * out.abs() + A * (4 * ds[:, None] + 2.0 ** -20 + u * u + chain)
    if half:
        tol = tol + 2.0 ** -25 * (n - lo) * v.abs().max()
    tol_lse = 2 * ds + 2.0 ** -20 + chain + 4 * F * lse.abs()
    return out, lse, tol, tol_lse


def check(q, c, ks, vs, window=0, scale=None, where="cpu", **kw):
    from nsa_amd.decode import dense_decode_step
    out, lse = dense_decode_step(q, c, scale=scale, sliding_window=window, return_lse=True, **kw)
    assert out.dtype == q.dtype and out.shape == (q.shape[0], q.shape[1], c.dv) and lse.shape == q.shape[:2]
    scale = q.shape[2] ** -0.5 if scale is None else scale
    got, got_lse = out.double().to(where), lse.double().to(where)
    for b in range(len(ks)):
        ref, ref_lse, tol, tol_lse = plain(q[b].to(where), ks[b], vs[b], scale, window)
        assert torch.isfinite(got[b]).all(), b
        assert ((got[b] - ref).abs() <= tol).all(), (b, len(ks[b]), float(((got[b] - ref).abs() / tol).max()))
        if len(ks[b]) == 0:
            assert (got[b] == 0).all() and (got_lse[b] == -math.inf).all()
        else:
            assert ((got_lse[b] - ref_lse).abs() <= tol_lse).all(), (b, len(ks[b]))
    return out, lse


LENS = [700, 0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 257, 1000, 2049]


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("dtype,hq,hkv,dk,dv", [
    (torch.bfloat16, 64, 4, 128, 128),
    (torch.float16, 24, 2, 192, 128),
    (torch.bfloat16, 8, 8, 64, 64),
    (torch.float32, 4, 1, 64, 64),
    (torch.float32, 16, 2, 128, 128),
    (torch.float32, 6, 1, 192, 128),
    (torch.float16, 4, 2, 32, 32),
])
@pytest.mark.parametrize("window", [0, 1, 100])
def test_every_length(paged, dtype, hq, hkv, dk, dv, window):
    c, ks, vs = make_cache(paged, LENS, 2112, hkv, dk, dv, dtype, seed=10)
    q = randn(len(LENS), hq, dk, seed=9, dtype=dtype).to(DEV)
    check(q, c, ks, vs, window)


@pytest.mark.parametrize("dtype,dk,dv", [(torch.bfloat16, 128, 128), (torch.float32, 64, 64), (torch.bfloat16, 192, 128),
                                         (torch.float32, 192, 128)])
@pytest.mark.parametrize("group", [1, 2, 3, 7, 15, 16, 17, 24, 32, 33, 48, 64, 65, 80, 130])
@pytest.mark.parametrize("cap", [320, 12800])          # beyond 1024 pages per call a group of up to 64 heads stays together
def test_every_group_size(cap, dtype, dk, dv, group):
    lens = [300, 77, 1]
    c, ks, vs = make_cache(True, lens, cap, 2, dk, dv, dtype, seed=30)
    q = randn(len(lens), 2 * group, dk, seed=29, dtype=dtype).to(DEV)
    check(q, c, ks, vs)


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("garbage", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_lies_behind_a_sequence_does_not_matter(paged, garbage, dtype):
    lens = [1, 5, 32, 40, 64, 70, 100, 0, 333]
    c, ks, vs = make_cache(paged, lens, 384, 2, 64, 64, dtype, seed=50, garbage=garbage)
    q = randn(len(lens), 8, 64, seed=49, dtype=dtype).to(DEV)
    check(q, c, ks, vs)
    # and what lies before the window
    for b, n in enumerate(lens):
        for j in range(max(0, n - 37)):
            if paged:
                c.k_pool[c.block_table[b, j // 64].long(), j % 64] = garbage
                c.v_pool_t[c.block_table[b, j // 64].long(), :, :, j % 64] = garbage
            else:
                c.k[b, j] = garbage
                c.vt[b, :, :, j] = garbage
    check(q, c, ks, vs, window=37)


@pytest.mark.parametrize("cap", [256, 2048])                      # one launch, and the split schedule
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nan_among_the_visible_comes_through(cap, dtype):
    """a NaN in a query is its head's, in a key all heads' that read it, in a value one channel's; nobody else's"""
    from nsa_amd.decode import dense_decode_step
    lens = [200, cap, 130]
    c, ks, vs = make_cache(True, lens, cap, 2, 64, 64, dtype, seed=55)
    q = randn(3, 8, 64, seed=56, dtype=dtype).to(DEV)
    want, want_lse = dense_decode_step(q, c, return_lse=True)
    bad = q.clone()
    bad[0, 1, 5] = math.nan
    page = c.block_table[1, 1].long()
    c.k_pool[page, 3, 1, 7] = math.nan
    c.v_pool_t[c.block_table[2, 0].long(), 0, 9, 2] = math.nan
    out, lse = dense_decode_step(bad, c, return_lse=True)
    nan, nan_lse = torch.zeros_like(out, dtype=torch.bool), torch.zeros_like(lse, dtype=torch.bool)
    nan[0, 1] = nan[1, 4:] = nan[2, :4, 9] = True
    nan_lse[0, 1] = nan_lse[1, 4:] = True
    assert torch.equal(out.isnan(), nan) and torch.equal(lse.isnan(), nan_lse)
    assert torch.equal(out[~nan], want[~nan]) and torch.equal(lse[~nan_lse], want_lse[~nan_lse])


def test_lowest_values_as_scores_and_large_scores():
    """Scores at the ends of the range: one key far above the others, and all of them equally low."""
    dtype = torch.float32
    lens = [200, 200]
    c, ks, vs = make_cache(True, lens, 256, 1, 64, 64, dtype, seed=60)
    q = randn(2, 4, 64, seed=61, dtype=dtype).to(DEV)
    for scale in (-0.125, 0.0, 30.0):
        check(q, c, ks, vs, scale=scale)


@pytest.mark.parametrize("paged", [True, False])
def test_many_sequences(paged):
    """more sequences than a wavefront has lanes, most of them empty or short, a few long"""
    g = random.Random(3)
    lens = [g.choice([0, 0, 1, 5, 64, 130]) for _ in range(203)]
    lens[70], lens[202] = 3000, 2500
    c, ks, vs = make_cache(paged, lens, 3008, 2, 64, 64, torch.bfloat16, seed=70)
    q = randn(len(lens), 16, 64, seed=69, dtype=torch.bfloat16).to(DEV)
    check(q, c, ks, vs)


@pytest.mark.parametrize("seed", range(30))
def test_random_shapes(seed):
    """batch, lengths, capacity, heads, types, windows and scales drawn together"""
    g = random.Random(1000 + seed)
    dtype = g.choice([torch.bfloat16, torch.float16, torch.float32])
    dk, dv = g.choice([(32, 32), (64, 64), (128, 128), (192, 128)])
    hkv, group = g.choice([1, 2, 3, 5, 8]), g.choice([1, 2, 5, 8, 16, 20, 33, 64, 70])
    B = g.choice([1, 2, 3, 9, 63, 64, 65, 130])
    cap = g.choice([64, 128, 320, 1024, 1088, 2048] if B > 10 else [64, 192, 1024, 2048, 5056])
    lens = [g.choice([g.randint(0, cap), cap, g.randint(0, min(cap, 130))]) for _ in range(B)]
    window = g.choice([0, 0, 0, 1, 63, 64, 65, g.randint(1, cap)])
    paged = g.random() < 0.6
    c, ks, vs = make_cache(paged, lens, cap, hkv, dk, dv, dtype, seed=2000 + 300 * seed, garbage=g.choice([None, math.nan]))
    q = randn(B, hkv * group, dk, seed=3000 + seed, dtype=dtype).to(DEV)
    if B > 10:                                             # the reference runs on the GPU for the many
        ks, vs = [k.to(DEV) for k in ks], [v.to(DEV) for v in vs]
    check(q, c, ks, vs, window, g.choice([None, None, 0.05, -0.2]), where=DEV if B > 10 else "cpu")


def test_units_of_more_pages_than_a_wavefront_has_lanes():
    """64 kv heads leave 16 units for 1500 pages, so a unit's page ids are read in several runs"""
    from nsa_amd.decode import NSAPagedDecodeCache, dense_decode_step
    H, D, n, dtype = 64, 32, 95_990, torch.bfloat16
    P = (n + 63) // 64
    c = NSAPagedDecodeCache(2, P + 1, n, H, D, D, dtype=dtype, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(4)
    c.k_pool.copy_(torch.randn(c.k_pool.shape, generator=gen, device=DEV, dtype=dtype))
    c.v_pool_t.copy_(torch.randn(c.v_pool_t.shape, generator=gen, device=DEV, dtype=dtype))
    order = torch.randperm(P, generator=torch.Generator().manual_seed(5)) + 1
    c.block_table[0, :P] = order.int().to(DEV)
    c.block_table[1, 0] = P + 1
    c.ctx_lens.copy_(torch.tensor([n, 50], dtype=torch.int32))
    q = torch.randn(2, H, D, generator=gen, device=DEV, dtype=dtype)
    out, lse = dense_decode_step(q, c, return_lse=True)
    for b, m in ((0, n), (1, 50)):
        ids = c.block_table[b, :(m + 63) // 64].long()
        for h in range(0, H, 9):
            k = c.k_pool[ids, :, h].reshape(-1, 1, D)[:m]
            v = c.v_pool_t[ids, h].transpose(1, 2).reshape(-1, 1, D)[:m]
            ref, ref_lse, tol, tol_lse = plain(q[b, h:h + 1], k, v, D ** -0.5, 0)
            assert ((out[b, h:h + 1].double() - ref).abs() <= tol).all()
            assert ((lse[b, h:h + 1].double() - ref_lse).abs() <= tol_lse).all()


def test_offsets_beyond_32_bits():
    """pages behind element 2^31 of both pools"""
    from nsa_amd.decode import NSAPagedDecodeCache, dense_decode_step
    H, D, dtype = 4, 128, torch.bfloat16
    pages = 2 ** 31 // (64 * H * D) + 40
    c = NSAPagedDecodeCache(1, pages, 2048, H, D, D, dtype=dtype, device=DEV)
    n = 32 * 64 - 11
    k = randn(2048, H, D, seed=80, dtype=dtype)
    v = randn(2048, H, D, seed=81, dtype=dtype)
    c.k_pool[pages - 31:] = k.view(32, 64, H, D).to(DEV)
    c.v_pool_t[pages - 31:] = v.view(32, 64, H, D).permute(0, 2, 3, 1).to(DEV)
    c.block_table[0] = torch.arange(pages - 31, pages + 1, dtype=torch.int32, device=DEV)
    c.ctx_lens.fill_(n)
    q = randn(1, 64, D, seed=82, dtype=dtype).to(DEV)
    check(q, c, [k[:n]], [v[:n]])


def test_lengths_and_page_ids_outside_the_cache_stay_inside_it():
    """a length beyond the capacity counts as the capacity, a negative one as 0; an id outside the pool reads page 0"""
    from nsa_amd.decode import dense_decode_step
    lens = [128, 128, 128]
    c, ks, vs = make_cache(True, lens, 128, 2, 64, 64, torch.bfloat16, seed=90)
    q = randn(3, 8, 64, seed=91, dtype=torch.bfloat16).to(DEV)
    want = dense_decode_step(q, c)
    c.ctx_lens.copy_(torch.tensor([129, 10 ** 6, -5], dtype=torch.int32))
    out, lse = dense_decode_step(q, c, return_lse=True)
    assert torch.equal(out[:2], want[:2]) and (out[2] == 0).all() and (lse[2] == -math.inf).all()
    c.ctx_lens.fill_(128)
    c.block_table[0, 1] = c.num_pages
    c.block_table[1, 1] = -1
    got = dense_decode_step(q, c)
    c.block_table[:2, 1] = 0
    assert torch.equal(got, dense_decode_step(q, c))


@pytest.mark.parametrize("window", [0, 200])
def test_equals_the_last_row_of_the_prefill_kernels(window):
    """the same token through sliding_window_attn, whose window covers the whole prompt or part of it"""
    import nsa_amd
    from nsa_amd.decode import NSADecodeCache, dense_decode_step
    T, hq, hkv, D, dtype = 777, 16, 2, 128, torch.bfloat16
    q, k, v = (randn(1, T, h, D, seed=100 + h, dtype=dtype).to(DEV) for h in (hq, hkv, hkv))
    rows = nsa_amd.sliding_window_attn(q, k, v, window or T)
    c = NSADecodeCache(1, T, hkv, D, D, dtype=dtype, device=DEV)
    c.fill(k, v)
    out = dense_decode_step(q[:, -1], c, sliding_window=window)
    u = torch.finfo(dtype).eps / 2      # both sides: probabilities and output rounded (|v| < 5, the weights sum to 1)
    assert float((out.double() - rows[:, -1].double()).abs().max()) <= 2 * u * (5 + float(rows.abs().max()))


def test_buffers_strides_and_streams():
    from nsa_amd.decode import dense_decode_step
    lens = [500, 3]
    c, ks, vs = make_cache(True, lens, 512, 2, 64, 64, torch.bfloat16, seed=110)
    wide = randn(2, 8, 3, 64, seed=111, dtype=torch.bfloat16).to(DEV)
    q = wide[:, :, 1]                                       # heads 3 * 64 apart
    want, want_lse = check(q, c, ks, vs)
    out = torch.full((2, 8, 64), 7.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((2, 8), 7.0, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = dense_decode_step(q, c, out=out, lse=lse)
        b = dense_decode_step(q, c)
    torch.cuda.current_stream().wait_stream(side)
    assert a is out and torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(b, want)
    assert torch.equal(dense_decode_step(q, c, sliding_window=2 ** 40), want)


def test_calls_on_two_streams_at_once_share_nothing():
    from nsa_amd.decode import dense_decode_step
    lens = [3000, 700, 4000, 1]
    c, ks, vs = make_cache(True, lens, 4032, 4, 128, 128, torch.bfloat16, seed=130)
    qs = [randn(4, 64, 128, seed=131 + i, dtype=torch.bfloat16).to(DEV) for i in range(2)]
    want = [check(q, c, ks, vs)[0] for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(dense_decode_step(qs[i], c))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_refusals():
    from nsa_amd.decode import dense_decode_step
    c, _, _ = make_cache(True, [500, 3], 512, 2, 64, 64, torch.bfloat16, seed=115)
    q = torch.zeros(2, 8, 64, dtype=torch.bfloat16, device=DEV)
    z = dict(dtype=torch.bfloat16, device=DEV)
    for bad in (dict(q=q[:1]), dict(q=q[0]), dict(q=q[..., :32]), dict(q=q.half()), dict(q=q[:, :7]), dict(q=q[:, :0]),
                dict(out=torch.empty(2, 8, 32, **z)), dict(out=torch.empty(2, 8, 64, device=DEV)), dict(out=q),
                dict(out=torch.empty(8, 2, 64, **z).transpose(0, 1)), dict(out=torch.empty(2 * 8 * 64 + 4, **z)[4:].view(2, 8, 64)),
                dict(lse=torch.empty(2, 8, **z)), dict(lse=torch.empty(2, 4, device=DEV)), dict(sliding_window=-1),
                dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            dense_decode_step(**dict(dict(q=q, cache=c), **bad))
    wide, _, _ = make_cache(True, [5], 64, 1, 96, 96, torch.bfloat16, seed=116)
    with pytest.raises(NotImplementedError):
        dense_decode_step(torch.zeros(1, 2, 96, **z), wide)


def test_captured_calls_follow_the_growing_cache():
    """two graphs captured over the same cache, replayed in turn while the sequences grow, equal the eager calls"""
    from nsa_amd.decode import NSAPagedDecodeCache, dense_decode_step
    B, hq, hkv, D, dtype, T0, steps = 3, 16, 2, 128, torch.bfloat16, 600, 70
    c = NSAPagedDecodeCache(B, 40, 768, hkv, D, D, dtype=dtype, device=DEV)
    k, v = (randn(B, T0 + steps, hkv, D, seed=120 + i, dtype=dtype).to(DEV) for i in range(2))
    q = randn(steps, B, hq, D, seed=122, dtype=dtype).to(DEV)
    c.fill(k[:, :T0], v[:, :T0])
    fixed = torch.zeros(B, hq, D, dtype=dtype, device=DEV)
    graphs, outs = [], []
    for window in (0, 100):
        dense_decode_step(fixed, c, sliding_window=window)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(dense_decode_step(fixed, c, sliding_window=window))
        graphs.append(g)
    for s in range(steps):
        c.append(k[:, T0 + s], v[:, T0 + s])
        fixed.copy_(q[s])
        for g, out, window in zip(graphs, outs, (0, 100)):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, dense_decode_step(q[s], c, sliding_window=window)), (s, window)
    for b in range(B):
        ref, _, tol, _ = plain(q[-1, b].cpu(), k[b].cpu(), v[b].cpu(), D ** -0.5, 0)
        assert ((outs[0][b].double().cpu() - ref).abs() <= tol).all()


@pytest.mark.parametrize("lens,cap,hq,hkv", [([1000, 997], 1024, 4, 1), ([2000] * 64, 2048, 8, 4), ([1500] * 40, 2048, 64, 1)])
def test_float16_keeps_what_lies_far_below_the_maximum(lens, cap, hq, hkv):
    """One key takes almost all of the weight and has a value of zero, so the output is the sum of the others' weights of
    e^-18.06 = 2^-26.06 each: below the last step of float16 beside a maximum of 1, and held beside one of 2^7.  A wavefront's
    probability is off by 2^-25 at most where float16 ends, the denominator then is at least 2^7 in the same units, hence
    2^-32 n max |v| in the place of the bound's last term."""
    from nsa_amd.decode import dense_decode_step
    dk = dv = 32
    c, ks, vs = make_cache(False, lens, cap, hkv, dk, dv, torch.float16, seed=140)
    for k, v in zip(ks, vs):
        k.zero_()
        k[0, :, 0] = 4.25
        v.fill_(1024.0)
        v[0] = 0.0
    for b, n in enumerate(lens):
        c.k[b, :n] = ks[b].to(DEV)
        c.vt[b, :, :, :n] = vs[b].permute(1, 2, 0).to(DEV)
    q = torch.zeros(len(lens), hq, dk, dtype=torch.float16)
    q[:, :, 0] = 4.25
    out, lse = dense_decode_step(q.to(DEV), c, scale=1.0, return_lse=True)
    for b, n in enumerate(lens):
        ref, ref_lse, tol, tol_lse = plain(q[b], ks[b], vs[b], 1.0, 0)
        tol = tol + (2.0 ** -32 - 2.0 ** -25) * n * 1024.0
        err = (out[b].double().cpu() - ref).abs()
        assert (err <= tol).all(), (b, float((err / tol).max()))
        assert ((lse[b].double().cpu() - ref_lse).abs() <= tol_lse).all()


def test_results_that_overlap_the_operands_are_refused():
    """out or lse inside another operand's memory, at its start or later; right behind it they may lie"""
    from nsa_amd.decode import dense_decode_step
    c, ks, vs = make_cache(True, [500, 3], 512, 2, 64, 64, torch.bfloat16, seed=117)
    n = 2 * 8 * 64
    pool = torch.zeros(4 * n, dtype=torch.bfloat16, device=DEV)
    q = pool[n:2 * n].view(2, 8, 64)
    q.copy_(randn(2, 8, 64, seed=118, dtype=torch.bfloat16))
    out_at = lambda i: pool[i:i + n].view(2, 8, 64)                                     # noqa: E731
    lse_at = lambda i: pool[i:i + 32].view(torch.float32).view(2, 8)                    # noqa: E731
    for bad in (dict(out=out_at(n)), dict(out=out_at(n + 8)), dict(out=out_at(8)), dict(out=out_at(2 * n - 8)),
                dict(lse=lse_at(n)), dict(lse=lse_at(2 * n - 32)), dict(out=out_at(2 * n), lse=lse_at(3 * n - 32)),
                dict(out=c.k_pool.view(-1)[-n:].view(2, 8, 64)), dict(out=c.v_pool_t.view(-1)[:n].view(2, 8, 64)),
                dict(lse=c.block_table.view(torch.float32).view(-1)[:16].view(2, 8))):
        with pytest.raises(ValueError, match="overlap"):
            dense_decode_step(q, c, **bad)
    want, _ = check(q, c, ks, vs)
    got, _ = check(q, c, ks, vs, out=out_at(2 * n), lse=lse_at(3 * n))
    assert torch.equal(got, want) and torch.equal(dense_decode_step(q, c, out=out_at(0)), want)


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("cap", [192, 2048])                      # one launch, and the split schedule
@pytest.mark.parametrize("dtype,group,dk,dv", [(torch.bfloat16, 4, 64, 64), (torch.float16, 4, 64, 64), (torch.float32, 4, 64, 64),
                                               (torch.bfloat16, 16, 128, 128), (torch.float16, 20, 32, 32),
                                               (torch.bfloat16, 64, 192, 128), (torch.float16, 40, 128, 128)])
def test_infinities_among_the_visible_values_come_through(paged, cap, dtype, group, dk, dv):
    """a value of infinity makes its channel infinite for the heads that read it, one of each sign no number; every other
    channel and the log-sum-exp keep their bits"""
    from nsa_amd.decode import dense_decode_step
    lens = [1, 190, cap, 64, 33]
    c, ks, vs = make_cache(paged, lens, cap, 2, dk, dv, dtype, seed=150)
    q = randn(len(lens), 2 * group, dk, seed=151, dtype=dtype).to(DEV)
    want, want_lse = dense_decode_step(q, c, return_lse=True)
    expect = want.clone()

    def put(b, h, chan, key, x):
        if paged:
            c.v_pool_t[c.block_table[b, key // 64].long(), h, chan, key % 64] = x
        else:
            c.vt[b, h, chan, key] = x

    for b, h, chan, puts in ((0, 0, 3, [(0, math.inf)]), (0, 1, dv - 1, [(0, -math.inf)]), (1, 0, 0, [(0, math.inf)]),
                             (1, 0, 17, [(189, -math.inf), (3, -math.inf)]), (1, 1, 5, [(70, math.inf), (71, -math.inf)]),
                             (2, 1, 9, [(cap - 1, math.inf)]), (2, 1, 10, [(5, -math.inf), (cap - 40, math.inf)]),
                             (2, 0, 11, [(31, math.nan), (32, math.inf)]), (4, 0, 20, [(32, -math.inf)])):
        for key, x in puts:
            put(b, h, chan, key, x)
        expect[b, h * group:(h + 1) * group, chan] = sum(x for _, x in puts)
    out, lse = dense_decode_step(q, c, return_lse=True)
    assert torch.equal(out.isnan(), expect.isnan()) and torch.equal(out.nan_to_num(0.5), expect.nan_to_num(0.5))
    assert torch.equal(lse, want_lse)
    # before a window they do not matter
    out, lse = dense_decode_step(q, c, sliding_window=1, return_lse=True)
    for b, n in enumerate(lens):
        hidden = [x for x in ((0, 0, 3), (0, 1, dv - 1)) if b == 0] + [x for x in ((2, 1, 9),) if b == 2] + \
            [x for x in ((1, 0, 17),) if b == 1] + [x for x in ((4, 0, 20),) if b == 4]
        finite = torch.ones(2 * group, dv, dtype=torch.bool, device=DEV)
        for _, h, chan in hidden:
            finite[h * group:(h + 1) * group, chan] = False
        assert torch.equal(out[b].isfinite(), finite), b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_an_infinity_far_below_the_maximum_counts(dtype):
    """weights of 2^-60 beside the largest: 0 in float16, but not the formula's"""
    from nsa_amd.decode import dense_decode_step
    lens = [200]
    c, ks, vs = make_cache(True, lens, 256, 1, 64, 64, dtype, seed=160)
    c.k_pool.zero_()
    c.k_pool[c.block_table[0, 1].long(), 0, 0, 0] = 1.0                          # key 64: 60 ln 2 above all others
    c.v_pool_t[c.block_table[0, 2].long(), 0, 7, 1] = -math.inf
    q = torch.zeros(1, 4, 64, dtype=dtype, device=DEV)
    q[:, :, 0] = 1.0
    out = dense_decode_step(q, c, scale=60 * math.log(2))
    assert (out[0, :, 7] == -math.inf).all()
    rest = [i for i in range(64) if i != 7]
    v = vs[0][64, 0, rest].double().to(DEV)                                      # all of the weight but 200 * 2^-60
    assert ((out[0, :, rest].double() - v).abs() <= 2.0 ** -21 * v.abs() + 2.0 ** -50).all()


@pytest.mark.parametrize("lens,big", [([300, 1, 40], 119), ([2048] * 63 + [2000], 116)])   # one launch; units of 4 pages and more
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_near_the_end_of_the_range_do_not_overflow(lens, big, dtype):
    """Values of 2^big under weights that rise by 2^7.9 after a wavefront's first keys: sum exp(s - m) |v| stays below
    n 2^big < 2^128, so the sums have to, whatever the reference of the exponentials."""
    from nsa_amd.decode import NSADecodeCache
    c = NSADecodeCache(len(lens), max(lens), 1, 64, 64, dtype=dtype, device=DEV)
    key = torch.arange(max(lens))
    high = key % 256 >= 128 if len(lens) > 3 else key >= 256
    k = torch.zeros(max(lens), 1, 64)
    k[high, 0, 0] = 5.46875                                                  # 7.89 ln 2
    v = torch.full((max(lens), 1, 64), 2.0 ** big)
    v[:, :, ::2] *= -1
    v[:, :, 5] = 1.0
    ks, vs = [k[:n].to(dtype) for n in lens], [v[:n].to(dtype) for n in lens]
    for b, n in enumerate(lens):
        c.k[b, :n] = ks[b].to(DEV)
        c.vt[b, :, :, :n] = vs[b].permute(1, 2, 0).to(DEV)
    c.ctx_lens.copy_(torch.tensor(lens, dtype=torch.int32))
    q = torch.zeros(len(lens), 4, 64, dtype=dtype, device=DEV)
    q[:, :, 0] = 1.0
    check(q, c, ks, vs, scale=1.0)


# ---- float16 at the bound its reference of 2^7 below the maximum allows: l is at least 2^7 where a probability is off by 2^-25
# at most (float16's last step), so the term is 2^-32 n max |v| instead of plain()'s 2^-25 n max |v|

def check_float16(q, c, ks, vs, window=0, scale=None):
    from nsa_amd.decode import dense_decode_step
    out, lse = dense_decode_step(q, c, scale=scale, sliding_window=window, return_lse=True)
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for b, (k, v) in enumerate(zip(ks, vs)):
        ref, ref_lse, tol, tol_lse = plain(q[b].cpu(), k, v, scale, window)
        if len(k) == 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        seen = v[max(0, len(v) - window):] if window else v
        tol = tol + (2.0 ** -32 - 2.0 ** -25) * len(seen) * float(seen.abs().max())
        err = (out[b].double().cpu() - ref).abs()
        assert (err <= tol).all(), (b, len(k), float((err / tol).max()))
        assert ((lse[b].double().cpu() - ref_lse).abs() <= tol_lse).all()


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("hq,hkv,dk,dv", [(24, 2, 192, 128), (16, 1, 128, 128), (40, 2, 64, 64), (128, 2, 128, 128), (4, 2, 32, 32)])
@pytest.mark.parametrize("window", [0, 100])
def test_float16_at_every_length_within_the_tight_bound(paged, hq, hkv, dk, dv, window):
    c, ks, vs = make_cache(paged, LENS, 2112, hkv, dk, dv, torch.float16, seed=170)
    q = randn(len(LENS), hq, dk, seed=171, dtype=torch.float16).to(DEV)
    check_float16(q, c, ks, vs, window)
    check_float16(q, c, ks, vs, window, scale=0.4)                 # scores over some 60 powers of two


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (192, 128)])
@pytest.mark.parametrize("lens,cap,hq,hkv", [([1000, 997], 1024, 4, 1), ([2000] * 30, 2048, 8, 4), ([1500] * 20, 2048, 64, 1),
                                             ([200, 130], 256, 20, 1)])
def test_float16_far_below_the_maximum_in_every_layout(paged, dk, dv, lens, cap, hq, hkv):
    """one key with nearly all of the weight and a value of 0, all others at 2^-26.06 of it with values of 1024"""
    c, ks, vs = make_cache(paged, lens, cap, hkv, dk, dv, torch.float16, seed=180)
    for k, v in zip(ks, vs):
        k.zero_()
        k[0, :, 0] = 4.25
        v.fill_(1024.0)
        v[0] = 0.0
    for b, n in enumerate(lens):
        for p in range((n + 63) // 64):
            m, at = min(64, n - 64 * p), slice(64 * p, min(n, 64 * p + 64))
            k, v = ks[b][at].to(DEV), vs[b][at].permute(1, 2, 0).to(DEV)
            if paged:
                page = c.block_table[b, p].long()
                c.k_pool[page, :m], c.v_pool_t[page, :, :, :m] = k, v
            else:
                c.k[b, at], c.vt[b, :, :, at] = k, v
    q = torch.zeros(len(lens), hq, dk, dtype=torch.float16, device=DEV)
    q[:, :, 0] = 4.25
    check_float16(q, c, ks, vs, scale=1.0)


@pytest.mark.parametrize("lens", [[2048] * 33, [2048] * 36, [8192] * 36, [8000] * 38, [4096] * 63, [64 * (130 - b) for b in range(60)],
                                  [8192] * 34 + [0] * 20, [8192 * 4] + [64] * 62, [640] * 50 + [8192] * 3])
def test_fewer_sequences_than_units_make_no_second_round(lens):
    """A workgroup per unit and kv head, one round of them: 1024 of 32 / 32 channels, so 64 units where 16 kv heads share the
    card.  The partial states in the workspace tell how many units the sequences of more than one were cut into."""
    from nsa_amd import _lib
    B, H, D, rows = len(lens), 16, 32, 16
    cap = (max(lens) + 63) // 64 * 64
    z = dict(dtype=torch.bfloat16, device=DEV)
    pages = cap // 64
    k, v = torch.zeros(pages + 1, 64, H, D, **z), torch.zeros(pages + 1, H, D, 64, **z)
    k.normal_()
    v.normal_()
    table = torch.arange(1, pages + 1, dtype=torch.int32, device=DEV).repeat(B, 1)         # all read the same pages
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q, out = torch.randn(B, H, D, **z), torch.empty(B, H, D, **z)
    lib = _lib.load()
    need = lib.nsa_dense_decode_workspace_bytes(B, H, H, D, D, cap, 0, 0)
    slots = need // (4 * rows * (D + 2))
    assert slots == (64 + B) * H
    ws = torch.full((need // 4,), math.nan, device=DEV)
    rc = lib.nsa_dense_decode_step(q.data_ptr(), k.data_ptr(), v.data_ptr(), table.data_ptr(), pages, pages + 1, ctx.data_ptr(),
                                   out.data_ptr(), None, B, H, H, D, D, cap, 0, D ** -0.5, 0, ws.data_ptr(), need,
                                   torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    written = ~ws[slots * rows * D:].view(slots, rows, 2)[:, 0, 0].isnan()
    units = int(written.sum()) / H
    assert units == int(units) and units <= 64
    for b in range(0, B, 7):                                   # and the result is the sequence's own, however it was cut
        n = lens[b]
        if n == 0:
            assert (out[b] == 0).all()
            continue
        kb, vb = k[1:].reshape(-1, H, D)[:n].cpu(), v[1:].permute(0, 3, 1, 2).reshape(-1, H, D)[:n].cpu()
        ref, _, tol, _ = plain(q[b].cpu(), kb, vb, D ** -0.5, 0)
        assert ((out[b].double().cpu() - ref).abs() <= tol).all(), b


@pytest.mark.parametrize("cap", [192, 2048])                      # one launch, and the split schedule
@pytest.mark.parametrize("dtype,group,dk,dv", [(torch.bfloat16, 4, 64, 64), (torch.float16, 20, 128, 128), (torch.float32, 4, 64, 64),
                                               (torch.bfloat16, 64, 192, 128)])
def test_infinities_among_the_visible_keys(cap, dtype, group, dk, dv):
    """a score of -inf takes its key out, one of +inf leaves no number, all of -inf leave nothing: out 0 and lse -inf"""
    from nsa_amd.decode import dense_decode_step
    lens = [1, 190, cap, 70]
    c, ks, vs = make_cache(True, lens, cap, 1, dk, dv, dtype, seed=190)
    for b, keys in ((0, [0]), (1, [5, 64, 189]), (2, [cap - 1]), (3, range(70))):
        for j in keys:
            ks[b][j, 0, 2] = math.inf
            c.k_pool[c.block_table[b, j // 64].long(), j % 64, 0, 2] = math.inf
    q = randn(len(lens), group, dk, seed=191, dtype=dtype)
    q[:, :, 2] = 1.0
    q[:, ::2, 2] = -1.0
    out, lse = (t.double().cpu() for t in dense_decode_step(q.to(DEV), c, return_lse=True))
    for b, n in enumerate(lens):
        assert out[b, 1::2].isnan().all() and not lse[b, 1::2].isfinite().any(), b
        if b in (0, 3):
            assert (out[b, ::2] == 0).all() and (lse[b, ::2] == -math.inf).all()
            continue
        seen = ks[b][:, 0, 2].isfinite()
        ref, ref_lse, tol, tol_lse = plain(q[b, ::2].contiguous(), ks[b][seen], vs[b][seen], dk ** -0.5, 0)
        assert ((out[b, ::2] - ref).abs() <= tol).all() and ((lse[b, ::2] - ref_lse).abs() <= tol_lse).all(), b
