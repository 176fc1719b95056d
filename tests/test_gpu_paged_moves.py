"""GPU tests of forks, reorders, cuts and compaction of the paged K/V cache.  Nothing here is computed: what a slot holds
after a move has to equal, bit for bit, what its parent held, and everything else has to stay as it was."""
import random

import pytest
import torch

from tests.util import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def cache_of(batch, pages, cap, hkv=2, dk=64, dv=64, dtype=torch.bfloat16, block=32, stride=16, seed=None):
    from nsa_amd.decode import NSAPagedDecodeCache
    c = NSAPagedDecodeCache(batch, pages, cap, hkv, dk, dv, block, stride, dtype, DEV)
    if seed is not None:
        random.Random(seed).shuffle(c._free)
    return c


def rows_of(c, n):
    return (n - c.block) // c.stride + 1 if n >= c.block else 0


def held(c, b):
    """k [n,Hkv,Dk], v [n,Hkv,Dv] and the compressed rows of slot b, read through the device's page table"""
    n = int(c.ctx_lens[b])
    assert n == c._lens[b]
    ids = c.block_table[b, :(n + 63) // 64].long()
    k = c.k_pool[ids].reshape(-1, c.hkv, c.dk)[:n].clone()
    v = c.v_pool_t[ids].permute(0, 3, 1, 2).reshape(-1, c.hkv, c.dv)[:n].clone()
    r = rows_of(c, n)
    return k, v, c.ck[b, :r].clone(), c.cvt[b, :, :, :r].clone()


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def cut_to(c, state, n):
    r = rows_of(c, n)
    return state[0][:n], state[1][:n], state[2][:r], state[3][..., :r]


def check_books(c):
    holders = [0] * c.num_pages
    for b in range(c.batch):
        pages = c._pages_of(b)
        assert c.block_table[b].tolist() == pages + [0] * (c.max_pages - len(pages))
        for p in pages:
            holders[p] += 1
        if c._lens[b] % 64:
            assert c._refs[pages[-1]] == 1
    assert holders == list(c._refs)
    assert sorted(c._free[i] for i in range(len(c._free))) == [p for p in range(1, c.num_pages) if not holders[p]]


def filled(lens, cap, pages=None, seed=0, **kw):
    B = len(lens)
    c = cache_of(B, pages or sum((n + 63) // 64 for n in lens) + B, cap, seed=seed, **kw)
    dtype = c.k_pool.dtype
    for b, n in enumerate(lens):
        if n:
            c.fill(randn(n, c.hkv, c.dk, seed=seed + 2 * b, dtype=dtype).to(DEV),
                   randn(n, c.hkv, c.dv, seed=seed + 2 * b + 1, dtype=dtype).to(DEV), seq=b)
    return c


KINDS = [dict(hkv=4, dk=128, dv=128), dict(hkv=2, dk=192, dv=128, dtype=torch.float16),
         dict(hkv=1, dk=64, dv=64, dtype=torch.float32), dict(hkv=3, dk=8, dv=24, dtype=torch.float16),
         dict(hkv=2, dk=64, dv=64, block=16, stride=8), dict(hkv=1, dk=64, dv=128, block=64, stride=16)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [0, 1, 31, 32, 63, 64, 65, 127, 128, 300, 1000])
def test_fork(kind, n):
    c = filled([n, 200, 0, 70, 5], 1024, **kind)
    before = [held(c, b) for b in range(5)]
    # columns and rows behind the compressed rows are not written
    marks = [randn(*c.ck.shape, seed=77).to(c.ck), randn(*c.cvt.shape, seed=78).to(c.cvt)]
    r = rows_of(c, n)
    for b in (1, 2, 4):
        c.ck[b, r:], c.cvt[b, :, :, r:] = marks[0][b, r:], marks[1][b, :, :, r:]
    free = c.free_pages
    c.fork(0, [2, 4, 1])
    for b in (0, 1, 2, 4):
        assert same(held(c, b), before[0]), b
    assert same(held(c, 3), before[3])
    for b in (1, 2, 4):
        assert torch.equal(c.ck[b, r:], marks[0][b, r:]) and torch.equal(c.cvt[b, :, :, r:], marks[1][b, :, :, r:])
    check_books(c)
    assert c.free_pages == free + 4 + 1 - (3 if n % 64 else 0)      # the pages of slots 1 and 4, less the copies
    for cut in {0, n // 2, max(n - 1, 0), n // 64 * 64}:
        c.fork(0, 3, length=cut)
        assert same(held(c, 3), cut_to(c, before[0], cut)) and same(held(c, 0), before[0])
        check_books(c)


@pytest.mark.parametrize("kind", KINDS[:4])
@pytest.mark.parametrize("batch", [2, 7, 33, 130])
def test_reorder(kind, batch):
    rng = random.Random(batch)
    lens = [rng.choice([0, 1, 33, 64, 100, 200, 256]) for _ in range(batch)]
    c = filled(lens, 256, pages=6 * batch, seed=3, **kind)
    for turn in range(4):
        before = [held(c, b) for b in range(batch)]
        parents = rng.sample(range(batch), batch) if turn % 2 else [rng.randrange(batch) for _ in range(batch)]
        if turn == 3:
            ring = rng.sample(range(batch), batch)
            for i, b in enumerate(ring):
                parents[b] = ring[(i + 1) % batch]
        c.reorder(parents if turn else torch.tensor(parents, device=DEV))
        for b, p in enumerate(parents):
            assert same(held(c, b), before[p]), (turn, b, p)
        check_books(c)


def test_a_fork_goes_its_own_way():
    """appending to forks writes into no shared page: every slot stays what a cache of its own would hold"""
    from nsa_amd.decode import dense_decode_step, nsa_decode_step
    B, T, steps, H, D, dtype = 4, 165, 100, 2, 64, torch.bfloat16
    k, v = (randn(T, H, D, seed=5 + i, dtype=dtype).to(DEV) for i in range(2))
    kn, vn = (randn(steps, B, H, D, seed=7 + i, dtype=dtype).to(DEV) for i in range(2))
    q = randn(B, 8, D, seed=9, dtype=dtype).to(DEV)
    shared, apart = cache_of(B, 24, 320, H, D, D, seed=1), cache_of(B, 24, 320, H, D, D, seed=2)
    shared.fill(k, v, seq=0)
    shared.fork(0, [1, 2, 3])
    for b in range(B):
        apart.fill(k, v, seq=b)
    assert shared.free_pages == 24 - 2 - 4 and apart.free_pages == 24 - 12
    for s in range(steps):
        shared.append(kn[s], vn[s])
        apart.append(kn[s], vn[s])
    for b in range(B):
        assert same(held(shared, b), held(apart, b))
    check_books(shared)
    a, ia = nsa_decode_step(q, shared, None, 64, 2, 32, return_indices=True)
    b, ib = nsa_decode_step(q, apart, None, 64, 2, 32, return_indices=True)
    assert torch.equal(a, b) and torch.equal(ia, ib)
    assert torch.equal(dense_decode_step(q, shared), dense_decode_step(q, apart))
    free = shared.free_pages
    shared.release(1)
    assert shared.free_pages == free + 3                            # its own pages, not the two it shared
    shared.fill(k[:70], v[:70], seq=0)
    assert same(held(shared, 2), held(apart, 2))
    check_books(shared)


@pytest.mark.parametrize("n", [0, 1, 63, 64, 65, 100, 128, 190, 200])
def test_truncate(n):
    """a cut inside a page that others share gets a page of its own; appending afterwards equals a fresh cache"""
    c = filled([200, 50], 320, pages=20)
    c.fork(0, 1)
    before = held(c, 0)
    c.truncate(1, n)
    assert same(held(c, 1), cut_to(c, before, n)) and same(held(c, 0), before)
    check_books(c)
    kn, vn = (randn(90, 2, 2, 64, seed=20 + i, dtype=torch.bfloat16).to(DEV) for i in range(2))
    for s in range(90):
        c.append(kn[s], vn[s])
    k, v = held(c, 1)[:2]
    assert torch.equal(k, torch.cat([before[0][:n], kn[:, 1]])) and torch.equal(v, torch.cat([before[1][:n], vn[:, 1]]))
    fresh = cache_of(1, 6, 320)
    fresh.fill(before[0][:n], before[1][:n], seq=0)
    for s in range(90):
        fresh.append(kn[s, 1:], vn[s, 1:])
    assert same(held(c, 1)[:2], held(fresh, 0)[:2])
    check_books(c)


@pytest.mark.parametrize("seed", range(8))
def test_random_runs(seed):
    """appends, fills, forks, reorders, cuts, releases and compactions one after the other, against the tokens every slot
    should hold"""
    rng = random.Random(seed)
    kind = KINDS[seed % 4]
    B = rng.choice([2, 5, 9, 20])
    c = cache_of(B, 5 * B, 320, seed=seed, **kind)
    dtype, n_new = c.k_pool.dtype, 0
    want = [(torch.zeros(0, c.hkv, c.dk, dtype=dtype, device=DEV), torch.zeros(0, c.hkv, c.dv, dtype=dtype, device=DEV))
            for _ in range(B)]

    def fresh(*shape):
        nonlocal n_new
        n_new += 1
        return randn(*shape, seed=10_000 * seed + n_new, dtype=dtype).to(DEV)

    for step in range(60):
        op = rng.choice(["append", "append", "fill", "fork", "reorder", "truncate", "release", "compact"])
        before = [held(c, b) for b in range(B)]
        try:
            if op == "append":
                for _ in range(rng.choice([1, 3, 40])):
                    kn, vn = fresh(B, c.hkv, c.dk), fresh(B, c.hkv, c.dv)
                    c.append(kn, vn)
                    want = [(torch.cat([k, kn[b:b + 1]]), torch.cat([v, vn[b:b + 1]])) for b, (k, v) in enumerate(want)]
            elif op == "fill":
                b, n = rng.randrange(B), rng.choice([1, 64, 100, 200])
                k, v = fresh(n, c.hkv, c.dk), fresh(n, c.hkv, c.dv)
                c.fill(k, v, seq=b)
                want[b] = (k, v)
            elif op == "fork":
                src = rng.randrange(B)
                dst = rng.sample([b for b in range(B) if b != src], rng.randint(1, B - 1))
                n = rng.choice([None, rng.randint(0, len(want[src][0]))])
                c.fork(src, dst, n)
                for b in dst:
                    want[b] = (want[src][0][:n], want[src][1][:n])
                    assert same(held(c, b), cut_to(c, before[src], len(want[src][0]) if n is None else n))
            elif op == "reorder":
                parents = rng.sample(range(B), B) if rng.random() < 0.5 else [rng.randrange(B) for _ in range(B)]
                c.reorder(parents)
                want = [want[p] for p in parents]
                for b, p in enumerate(parents):
                    assert same(held(c, b), before[p])
            elif op == "truncate":
                b = rng.randrange(B)
                n = rng.randint(0, len(want[b][0]))
                c.truncate(b, n)
                want[b] = (want[b][0][:n], want[b][1][:n])
                assert same(held(c, b), cut_to(c, before[b], n))
            elif op == "release":
                b = rng.randrange(B)
                c.release(b)
                want[b] = (want[b][0][:0], want[b][1][:0])
            else:
                c.compact()
        except RuntimeError as e:
            assert "exhausted" in str(e) or "capacity" in str(e)
        for b in range(B):
            assert same(held(c, b)[:2], want[b]), (step, op, b)
        check_books(c)


def test_exhausted_pool_changes_nothing():
    c = filled([100, 100, 0, 0], 128, pages=5)
    before = [held(c, b) for b in range(4)]
    tensors = [t.clone() for t in (c.k_pool, c.v_pool_t, c.block_table, c.ck, c.cvt, c.ctx_lens)]
    for call in (lambda: c.fork(0, [2, 3]), lambda: c.reorder([0, 1, 0, 1])):
        with pytest.raises(RuntimeError, match="exhausted"):
            call()
        for t, u in zip(tensors, (c.k_pool, c.v_pool_t, c.block_table, c.ck, c.cvt, c.ctx_lens)):
            assert torch.equal(t, u)
        check_books(c)
    c.fork(0, 2)
    c.reorder([2, 2, 1, 3])                                         # slot 0's page becomes one of the copies
    assert same(held(c, 0), before[0]) and same(held(c, 1), before[0]) and same(held(c, 2), before[1])
    check_books(c)


def test_refilling_slots_that_share_pages():
    """the pool is just large enough once every holder of the shared pages lets go"""
    c = filled([256, 0, 0, 0], 256, pages=16)
    c.fork(0, [1, 2, 3])
    assert c.free_pages == 12
    k, v = (randn(4, 256, 2, 64, seed=30 + i, dtype=torch.bfloat16).to(DEV) for i in range(2))
    c.fill(k, v)
    assert c.free_pages == 0
    for b in range(4):
        assert torch.equal(held(c, b)[0], k[b]) and torch.equal(held(c, b)[1], v[b])
    check_books(c)
    c.fork(0, 1)
    with pytest.raises(RuntimeError, match="exhausted"):
        c.fill(torch.cat([k[0], k[0, :1]]).expand(4, -1, -1, -1)[:, :257], torch.cat([v[0], v[0, :1]]).expand(4, -1, -1, -1))
    check_books(c)


@pytest.mark.parametrize("kind", KINDS[:4])
def test_compact(kind):
    """more moved pages than one launch takes"""
    lens = [64 * 130, 64 * 120 + 7, 64 * 300 + 1, 0, 64 * 250]
    c = filled(lens, 64 * 310, pages=1700, seed=4, **kind)
    c.fork(2, 3)
    c.release(0)
    before = [held(c, b) for b in range(5)]
    used = c.num_pages - 1 - c.free_pages
    high = sum(p > used for b in range(5) for p in set(c._pages_of(b)))
    assert high > 384
    assert c.compact() == used
    for b in range(5):
        assert same(held(c, b), before[b])
        assert all(1 <= p <= used for p in c._pages_of(b))
    check_books(c)
    assert c.compact() == used and c._free[-1] == used + 1


def test_pages_behind_element_two_to_the_31():
    c = cache_of(3, 2 ** 31 // (64 * 4 * 128) + 60, 512, 4, 128, 128)
    n = len(c._free)
    for i in range(n // 2):                                         # the highest pages first
        c._free[i], c._free[n - 1 - i] = c._free[n - 1 - i], c._free[i]
    k, v = (randn(300, 4, 128, seed=40 + i, dtype=torch.bfloat16).to(DEV) for i in range(2))
    c.fill(k, v, seq=0)
    assert min(c._pages_of(0)) * 64 * 4 * 128 > 2 ** 31
    c.fork(0, [1, 2])
    c.truncate(2, 100)
    for b, m in ((0, 300), (1, 300), (2, 100)):
        got = held(c, b)
        assert torch.equal(got[0], k[:m]) and torch.equal(got[1], v[:m])
    assert c.compact() == 5 + 1 + 1
    for b, m in ((0, 300), (1, 300), (2, 100)):
        got = held(c, b)
        assert torch.equal(got[0], k[:m]) and torch.equal(got[1], v[:m])
    check_books(c)


def test_moves_beside_captured_decode_steps():
    """a decode graph captured before the moves goes on over the moved sequences; a move itself cannot be captured"""
    from nsa_amd.decode import NSADecodeGraph, dense_decode_step, nsa_decode_step
    B, T, H, D, dtype = 3, 150, 2, 64, torch.bfloat16
    ca, cb = (filled([T] * B, 512, pages=40, seed=6) for _ in range(2))
    graph = NSADecodeGraph(ca, 8, 64, 2, 32, use_gates=False)
    dense_q = torch.zeros(B, 8, D, dtype=dtype, device=DEV)
    dense_decode_step(dense_q, ca)
    dense = torch.cuda.CUDAGraph()
    with torch.cuda.graph(dense):
        dense_out = dense_decode_step(dense_q, ca)
    for s in range(30):
        q, kn, vn = (randn(B, h, D, seed=50 + 3 * s + i, dtype=dtype).to(DEV) for i, h in enumerate((8, H, H)))
        out = graph.step(q, kn, vn)
        cb.append(kn, vn)
        assert torch.equal(out, nsa_decode_step(q, cb, None, 64, 2, 32)), s
        dense_q.copy_(q)
        dense.replay()
        assert torch.equal(dense_out, dense_decode_step(q, cb)), s
        if s % 7 == 3:
            for c in (ca, cb):
                c.reorder([2, 0, 0])
                c.truncate(1, c._lens[1] - 5)
        if s == 20:
            ca.compact()
    for b in range(B):
        assert same(held(ca, b), held(cb, b))
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ca.fork(0, 1)
    check_books(ca)


def test_a_stream_of_its_own():
    c = filled([200, 0, 0], 256, pages=12)
    before = held(c, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.fork(0, [1, 2])
        c.truncate(1, 100)
        c.reorder([1, 0, 2])
    torch.cuda.current_stream().wait_stream(side)
    assert same(held(c, 0), cut_to(c, before, 100)) and same(held(c, 1), before) and same(held(c, 2), before)


def test_sampling_from_a_prompt_with_pictures():
    """Used together: a layer with positions on three axes reads a prompt into the cache, the prompt is forked for several
    samples, each goes on token by token, the samples change places, take tokens back, and the cache is compacted; a
    second run without forks, every sample on its own, gives the same outputs bit for bit."""
    from nsa_amd.decode import NSAPagedDecodeCache, dense_decode_step
    from nsa_amd.layer import NSAAttentionLayer
    torch.manual_seed(0)
    layer = NSAAttentionLayer(256, 8, 2, 64, rope_dim=32, compressor_mode="mean", gate_activation="sigmoid",
                              selected_block_count=4, sliding_window=64, rope_axes=(4, 6, 6), device=DEV,
                              dtype=torch.bfloat16)
    T, B, steps = 140, 3, 70
    grid = torch.arange(T, device=DEV)
    pos = torch.stack([torch.clamp(grid, max=40), grid % 12, grid // 12]).view(3, 1, T)
    prompt = randn(1, T, 256, seed=60, scale=0.5, dtype=torch.bfloat16).to(DEV)
    tokens = randn(steps, B, 1, 256, seed=61, scale=0.5, dtype=torch.bfloat16).to(DEV)
    queries = randn(steps, B, 8, 64, seed=62, dtype=torch.bfloat16).to(DEV)
    shared = NSAPagedDecodeCache(B, 30, 512, 2, 64, 64, device=DEV)
    apart = NSAPagedDecodeCache(B, 30, 512, 2, 64, 64, device=DEV)
    first = NSAPagedDecodeCache(1, 10, 512, 2, 64, 64, device=DEV)
    with torch.no_grad():
        layer(prompt, position_ids=pos, past_key_value=first)
        k, v = held(first, 0)[:2]
        shared.fill(k, v, seq=0)
        shared.fork(0, [1, 2])
        for b in range(B):
            apart.fill(k, v, seq=b)
        histories = [[] for _ in range(B)]
        for s in range(steps):
            place = torch.full((3, B), 200 + s, device=DEV)
            outs = [layer(tokens[s], position_ids=place, past_key_value=c)[0] for c in (shared, apart)]
            dense = [dense_decode_step(queries[s], c) for c in (shared, apart)]
            assert torch.equal(*outs) and torch.equal(*dense), s
            for b in range(B):
                histories[b].append([t[-1:] for t in held(apart, b)[:2]])
            if s in (20, 50):                                       # two samples go on from the same one
                shared.reorder([1, 1, 0])
                histories = [list(histories[p]) for p in (1, 1, 0)]
                for b in range(B):
                    apart.fill(torch.cat([k] + [h[0] for h in histories[b]]), torch.cat([v] + [h[1] for h in histories[b]]),
                               seq=b)
                # the compressed rows of a fill and of appends are rounded from sums in another order
                for b in range(B):
                    apart.ck[b], apart.cvt[b] = shared.ck[b], shared.cvt[b]
            if s == 35:
                shared.truncate(2, T + 30)
                histories[2] = histories[2][:30]
                apart.fill(torch.cat([k] + [h[0] for h in histories[2]]), torch.cat([v] + [h[1] for h in histories[2]]), seq=2)
                apart.ck[2], apart.cvt[2] = shared.ck[2], shared.cvt[2]
                shared.compact()
    check_books(shared)
    assert shared.free_pages > apart.free_pages


class FailingLibrary:
    """The library with one function that fails before it does anything."""

    def __init__(self, lib, name):
        self.lib, self.name = lib, name

    def __getattr__(self, name):
        return (lambda *a: -4) if name == self.name else getattr(self.lib, name)


@pytest.mark.parametrize("name", ["nsa_paged_cache_move", "nsa_paged_cache_compact_move"])
def test_a_cache_whose_device_half_failed_takes_no_more_calls(name, monkeypatch):
    """the page table of the host is then ahead of the device's, so nothing may be built on it; reading goes on"""
    from nsa_amd import _lib
    from nsa_amd.decode import dense_decode_step
    c = filled([100, 130, 64], 256)
    c.truncate(0, 30)
    k, v = randn(3, 2, 64, seed=1, dtype=torch.bfloat16).to(DEV), randn(3, 2, 64, seed=2, dtype=torch.bfloat16).to(DEV)
    q = randn(3, 4, 64, seed=3, dtype=torch.bfloat16).to(DEV)
    want, tables = dense_decode_step(q, c), [t.clone() for t in (c.block_table, c.ctx_lens, c.k_pool, c.v_pool_t, c.ck, c.cvt)]
    lib = _lib.load()
    with monkeypatch.context() as m:
        m.setattr(_lib, "load", lambda: FailingLibrary(lib, name))
        with pytest.raises(RuntimeError, match="failed"):
            c.compact() if "compact" in name else c.reorder([1, 2, 0])
    for call in (lambda: c.fork(0, 1), lambda: c.reorder([0, 0, 1]), lambda: c.truncate(1, 5), lambda: c.release(1),
                 lambda: c.compact(), lambda: c.append(k, v), lambda: c.reserve_next(),
                 lambda: c.fill(k.expand(70, -1, -1, -1)[:, 0].contiguous(), v.expand(70, -1, -1, -1)[:, 0].contiguous(), seq=2)):
        with pytest.raises(RuntimeError, match="build a new"):
            call()
    assert same(tables, [c.block_table, c.ctx_lens, c.k_pool, c.v_pool_t, c.ck, c.cvt])
    assert torch.equal(dense_decode_step(q, c), want)
