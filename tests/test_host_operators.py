"""CPU-side checks of dense decode attention, the paged cache's forks and moves, and the rotation on several axes: refusals
and host bookkeeping (no kernel is launched here)."""
import ctypes
import os

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nsa_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from nsa_amd import build
        build.build()
    return _lib.load()


def test_dense_decode_argument_errors_do_not_launch(lib):
    """every call is refused before a launch (the pointers are not device memory)"""
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    names = ["q", "k", "v", "table", "max_pages", "num_pages", "lens", "out", "lse", "batch", "hq", "hkv", "dk", "dv", "cap",
             "window", "scale", "dtype", "ws", "ws_bytes", "stream"]
    good = dict(q=p, k=p, v=p, table=p, max_pages=64, num_pages=8, lens=p, out=p, lse=None, batch=2, hq=16, hkv=2, dk=64, dv=64,
                cap=0, window=0, scale=0.1, dtype=0, ws=p, ws_bytes=1 << 40, stream=None)

    def call(**kw):
        return lib.nsa_dense_decode_step(*[dict(good, **kw)[n] for n in names])

    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(lens=None), dict(out=None), dict(dtype=7), dict(batch=0),
                dict(hq=15), dict(hkv=0), dict(window=-1), dict(max_pages=0), dict(num_pages=0), dict(max_pages=1 << 30),
                dict(table=None, cap=0), dict(table=None, cap=100), dict(scale=float("inf")), dict(scale=float("nan")),
                dict(q=p + 2), dict(out=p + 8), dict(ws=None), dict(ws=p + 4), dict(ws_bytes=100),
                dict(batch=1 << 30, max_pages=1 << 20)):
        assert call(**bad) == -1, bad
        assert lib.nsa_last_error_string()
    for bad in (dict(dk=128), dict(dk=96, dv=96), dict(dk=192, dv=192)):
        assert call(**bad) == -2, bad
    assert lib.nsa_dense_decode_workspace_bytes(2, 16, 2, 64, 64, 128, 0, 0) == 0          # one unit per sequence
    assert lib.nsa_dense_decode_workspace_bytes(2, 16, 2, 64, 64, 4096, 64, 0) == 0        # a window of two pages at most
    assert lib.nsa_dense_decode_workspace_bytes(2, 16, 2, 64, 64, 4096, 0, 0) > 0
    assert lib.nsa_dense_decode_workspace_bytes(2, 15, 2, 64, 64, 4096, 0, 0) == -1
    assert lib.nsa_dense_decode_workspace_bytes(2, 16, 2, 64, 64, 100, 0, 0) == -1


def test_dense_decode_python_checks():
    from nsa_amd.decode import NSAPagedDecodeCache, dense_decode_step
    c = NSAPagedDecodeCache(2, 4, 128, 2, 64, 64, device="cpu")
    with pytest.raises(RuntimeError, match="GPU only"):
        dense_decode_step(torch.zeros(2, 4, 64, dtype=torch.bfloat16), c)


def test_rope_axes_argument_errors_do_not_launch(lib):
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    names = ["packed", "q", "k", "v", "gates", "inv", "pos", "axes", "pair_axis", "total", "ld", "q_off", "k_off", "v_off",
             "g_off", "hq", "hkv", "dk", "dv", "rope_off", "rope_dim", "interleaved", "pack", "dtype", "stream"]
    pairs = lambda *a: (ctypes.c_int32 * 128)(*a)                                       # noqa: E731
    good = dict(packed=p, q=p, k=p, v=p, gates=p, inv=p, pos=p, axes=3, pair_axis=pairs(0, 1, 2), total=4, ld=416, q_off=0,
                k_off=256, v_off=320, g_off=384, hq=4, hkv=1, dk=64, dv=64, rope_off=0, rope_dim=32, interleaved=0, pack=0,
                dtype=0, stream=None)

    def call(**kw):
        return lib.nsa_qkv_rope_axes(*[dict(good, **kw)[n] for n in names])

    for bad in (dict(packed=None), dict(q=None), dict(inv=None), dict(pos=None), dict(pair_axis=None), dict(dtype=3),
                dict(total=0), dict(dk=60), dict(ld=412), dict(k_off=252), dict(v_off=400), dict(g_off=405), dict(q_off=-8),
                dict(rope_dim=24), dict(rope_dim=0), dict(rope_off=40), dict(rope_off=4), dict(axes=0), dict(axes=5),
                dict(axes=2), dict(pair_axis=pairs(-1)), dict(packed=p + 4), dict(hq=1 << 26)):
        assert call(**bad) == -1, bad
        assert lib.nsa_last_error_string()
    assert call(pack=1, k_off=248) == -1 and call(pack=1, g_off=380) == -1              # ranges of a packed row overlap
    assert call(dk=512, rope_dim=512, ld=8192, k_off=2048, v_off=4096, g_off=6000) == -2


def test_rope_pair_axes_and_the_layers_checks():
    from nsa_amd.layer import NSAAttentionLayer, rope_pair_axes
    assert rope_pair_axes((2, 3, 1)) == (0, 0, 1, 1, 1, 2)
    assert rope_pair_axes((2, 3, 1), "turns") == (0, 1, 2, 0, 1, 1)
    assert rope_pair_axes((4,)) == (0, 0, 0, 0) and rope_pair_axes((0, 2)) == (1, 1)
    for bad in (((), "blocks"), ((1,) * 5, "blocks"), ((-1, 2), "blocks"), ((1, 2), "rows")):
        with pytest.raises(ValueError):
            rope_pair_axes(*bad)
    for bad in (dict(rope_axes=(4, 6, 5)), dict(rope_axes=(4, 6, 6), rope_axes_spectrum="half"),
                dict(rope_axes=(4, 6, 6), rope_axes_layout="rows")):
        with pytest.raises(ValueError):
            NSAAttentionLayer(64, 2, 1, 64, rope_dim=32, **bad)
    with pytest.raises(ValueError):
        NSAAttentionLayer(64, 2, 1, 64, rope_dim=0, rope_axes=(0,))
    plain, own = (NSAAttentionLayer(64, 2, 1, 64, rope_dim=32, rope_axes=(4, 6, 6), rope_axes_spectrum=s)
                  for s in ("shared", "own"))
    assert torch.equal(plain.inv_freq, NSAAttentionLayer(64, 2, 1, 64, rope_dim=32).inv_freq)
    for lo, n in ((0, 4), (4, 6), (10, 6)):
        assert torch.allclose(own.inv_freq[lo:lo + n], 10000.0 ** -(torch.arange(n) / n), rtol=1e-6)
    cu = torch.tensor([0, 3, 3, 7], dtype=torch.int32)
    assert plain._axis_positions(None, 7, cu).tolist() == [[0, 1, 2, 0, 1, 2, 3]] * 3
    ids = torch.arange(42).view(3, 2, 7)
    assert torch.equal(plain._axis_positions(ids, 14, None), ids.reshape(3, 14))
    for bad in (torch.zeros(14), torch.zeros(2, 14), torch.zeros(3, 13)):
        with pytest.raises(ValueError, match="position_ids"):
            plain._axis_positions(bad, 14, None)


def test_rope_axes_python_checks(monkeypatch):
    """refusals of the tensor-level wrapper, on CPU tensors with the device check out of the way"""
    from nsa_amd import ops
    x = torch.zeros(3, 416, dtype=torch.bfloat16)
    args = (4, 1, 64, 64, (0, 256, 320, 384))
    good = dict(inv_freq=torch.zeros(16), positions=torch.zeros(3, 3, dtype=torch.int32), rope_off=0, rope_dim=32,
                pair_axis=[0, 1] * 8)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.qkv_rope_split(x, *args, **good)
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    for bad, err in ((dict(inv_freq=None), ValueError), (dict(positions=None), ValueError),
                     (dict(inv_freq=torch.zeros(8)), ValueError), (dict(pair_axis=[0] * 15), ValueError),
                     (dict(pair_axis=[3] * 16), ValueError), (dict(pair_axis=[-1] * 16), ValueError),
                     (dict(positions=torch.zeros(3, dtype=torch.int32)), ValueError),
                     (dict(positions=torch.zeros(3, 4, dtype=torch.int32)), ValueError),
                     (dict(positions=torch.zeros(5, 3, dtype=torch.int32)), ValueError),
                     (dict(positions=torch.zeros(3, 3)), TypeError)):
        with pytest.raises(err):
            ops.qkv_rope_split(x, *args, **dict(good, **bad))
    dq, dk, dv, dg = (torch.zeros(3, h, d, dtype=torch.bfloat16) for h, d in ((4, 64), (1, 64), (1, 64), (4, 3)))
    for bad in ((dq, dk[:2], dv, dg), (dq, dk, dv, dg.float()), (dq, dk[:, :, :32].contiguous(), dv, dg)):
        with pytest.raises(ValueError, match="agree"):
            ops.qkv_rope_pack(*bad, 416, args[4], **good)


# ------------------------------------------------------------------------------- forks and moves in the paged cache

class Model:
    """Every slot's tokens as a plain list; the cache's tensors hold token ids (one head, one channel group), its compressed
    rows the id of their last token."""

    def __init__(self, cache):
        self.c, self.next = cache, 1
        self.tokens = [[] for _ in range(cache.batch)]

    def append(self, b, n):
        c = self.c
        entries = c._grow(b, c._lens[b] + n)
        c._publish([(b, s, p) for s, p in entries])
        for _ in range(n):
            at = c._lens[b]
            page = c._pages_of(b)[at // 64]
            assert c._refs[page] == 1                       # a shared page is never written
            c.k_pool[page, at % 64] = c.v_pool_t[page, :, :, at % 64] = self.next
            self.tokens[b].append(self.next)
            c._lens[b] = at + 1
            if at + 1 >= c.block and (at + 1 - c.block) % c.stride == 0:
                row = (at + 1 - c.block) // c.stride
                c.ck[b, row] = c.cvt[b, :, :, row] = self.next
            self.next += 1
        c.ctx_lens[b] = c._lens[b]

    def check(self):
        c = self.c
        holders = [0] * c.num_pages
        for b, want in enumerate(self.tokens):
            n, pages = len(want), c._pages_of(b)
            assert c._lens[b] == n and int(c.ctx_lens[b]) == n and len(pages) == (n + 63) // 64
            assert c.block_table[b].tolist() == pages + [0] * (c.max_pages - len(pages))
            assert c._table[b * c.max_pages:(b + 1) * c.max_pages] == c.block_table[b].tolist()
            for p in pages:
                assert 0 < p < c.num_pages
                holders[p] += 1
            if n:
                ids = torch.tensor(pages)
                assert c.k_pool[ids].reshape(-1, c.hkv * c.dk)[:n, 0].tolist() == want
                assert c.v_pool_t[ids].permute(0, 3, 1, 2).reshape(-1, c.hkv * c.dv)[:n, -1].tolist() == want
            rows = (n - c.block) // c.stride + 1 if n >= c.block else 0
            last = [want[r * c.stride + c.block - 1] for r in range(rows)]
            assert c.ck[b, :rows, 0, 0].tolist() == last and c.cvt[b, 0, 0, :rows].tolist() == last
            if n % 64:
                assert c._refs[pages[-1]] == 1
        assert holders == list(c._refs)
        free = [c._free[i] for i in range(len(c._free))]
        assert sorted(free) == [p for p in range(1, c.num_pages) if holders[p] == 0]


def carry_out(c, moves):
    """The device half on CPU tensors, in the rounds of the kernel: the loads of a round before its stores."""
    rows = lambda n: min((n - c.block) // c.stride + 1, c.nc_cap) if n >= c.block else 0     # noqa: E731
    kept, i = None, 0
    while i < len(moves):
        cnt = 1
        while cnt < 8 and i + cnt < len(moves) and moves[i + cnt][1] >= 0:
            cnt += 1
        loaded = [None if m[0] < 0 else (c.ck[m[0]].clone(), c.cvt[m[0]].clone(), c.block_table[m[0]].clone())
                  for m in moves[i:i + cnt]]
        for (src, dst, n, tail_src, tail), val in zip(moves[i:i + cnt], loaded):
            if dst < 0:
                kept = val
                continue
            ck, cvt, table = kept if src < 0 else val
            if src != dst:
                c.ck[dst, :rows(n)] = ck[:rows(n)]
                c.cvt[dst, :, :, :rows(n)] = cvt[:, :, :rows(n)]
            table = table.clone()
            table[n // 64:] = 0
            if n % 64:
                table[n // 64] = tail
            c.block_table[dst] = table
            c.ctx_lens[dst] = n
        i += cnt
    for src, dst, n, tail_src, tail in moves:
        if n % 64 and dst >= 0 and tail_src != tail:
            c.k_pool[tail], c.v_pool_t[tail] = c.k_pool[tail_src].clone(), c.v_pool_t[tail_src].clone()


def plan(lib, c, slots, parents, lengths):
    n = len(slots)
    ints = ctypes.c_int32 * max(n, 1)
    moves, count = (ctypes.c_int32 * (10 * n + 10))(), ctypes.c_int32()
    rc = lib.nsa_paged_cache_plan(c._table, c._lens, c._held, c._refs, c._free.ids, ctypes.byref(c._free.n), c.batch,
                                  c.max_pages, c.num_pages, ints(*slots), ints(*parents), ints(*lengths), n, moves,
                                  ctypes.byref(count))
    if rc:
        return rc, None
    assert count.value <= 2 * n + 2
    return rc, [tuple(moves[5 * i:5 * i + 5]) for i in range(count.value)]


def small_cache(batch, pages, cap=320):
    from nsa_amd.decode import NSAPagedDecodeCache
    return NSAPagedDecodeCache(batch, pages, cap, 1, 8, 8, dtype=torch.float32, device="cpu")


def books(c):
    return (list(c._table), list(c._lens), list(c._held), list(c._refs), len(c._free),
            [c._free[i] for i in range(len(c._free))])


@pytest.mark.parametrize("seed", range(12))
def test_paged_moves_against_a_model(lib, seed):
    """random appends, forks, reorders, cuts and releases: tokens, compressed rows, page table, counts and free list"""
    import random
    rng = random.Random(seed)
    batch = rng.choice([2, 3, 5, 9, 17])
    c = small_cache(batch, rng.choice([batch * 2, batch * 5]))
    m = Model(c)
    refused = 0
    for _ in range(60):
        kind = rng.choice(["append", "append", "fork", "reorder", "assign", "truncate", "release"])
        if kind == "append":
            b, n = rng.randrange(batch), rng.choice([1, 2, 31, 33, 64, 100])
            need = (len(m.tokens[b]) + n + 63) // 64
            if need <= c.max_pages and need - c._held[b] <= len(c._free):
                m.append(b, n)
        elif kind == "release":
            b = rng.randrange(batch)
            c.release(b)
            m.tokens[b] = []
        else:
            if kind == "fork":
                src = rng.randrange(batch)
                slots = rng.sample([b for b in range(batch) if b != src], rng.randint(1, batch - 1))
                cut = rng.choice([len(m.tokens[src]), rng.randint(0, len(m.tokens[src]))])
                parents, lengths = [src] * len(slots), [cut] * len(slots)
            elif kind == "reorder":
                slots = list(range(batch))
                parents = rng.sample(slots, batch) if rng.random() < 0.5 else [rng.randrange(batch) for _ in slots]
                lengths = [rng.choice([-1, len(m.tokens[p])]) for p in parents]
            elif kind == "assign":
                slots = rng.sample(range(batch), rng.randint(1, batch))
                parents = [rng.randrange(batch) for _ in slots]
                lengths = [rng.randint(0, len(m.tokens[p])) for p in parents]
            else:
                slots = parents = [rng.randrange(batch)]
                lengths = [rng.randint(0, len(m.tokens[slots[0]]))]
            before = books(c)
            rc, moves = plan(lib, c, slots, parents, lengths)
            if rc:
                assert rc == -3 and books(c) == before
                refused += 1
            else:
                carry_out(c, moves)
                old = [list(t) for t in m.tokens]
                for s, p, n in zip(slots, parents, lengths):
                    m.tokens[s] = old[p][:n] if n >= 0 else list(old[p])
        m.check()
    assert refused < 40


@pytest.mark.parametrize("n", [2, 3, 62, 63, 64, 65, 66, 130, 200])
def test_paged_moves_in_cycles_of_any_length(lib, n):
    """all slots change places in one cycle, in two, and in one with branches"""
    for pattern in range(3):
        c = small_cache(n, 4 * n, cap=128)
        m = Model(c)
        for b in range(n):
            m.append(b, 40 + b % 60)
        order = torch.randperm(n, generator=torch.Generator().manual_seed(n + pattern)).tolist()
        parents = list(range(n))
        cut = n if pattern != 1 else max(2, n // 3)
        for lo, hi in ((0, cut), (cut, n)):
            ring = order[lo:hi]
            for i, b in enumerate(ring):
                parents[b] = ring[(i + 1) % len(ring)]
        if pattern == 2 and n > 5:
            parents[order[1]] = order[4]                     # order[2] and order[3] are left with one reader less
        rc, moves = plan(lib, c, list(range(n)), parents, [len(m.tokens[p]) for p in parents])
        assert rc == 0
        # a cycle's piece stays short enough for one launch
        start = None
        for i, mv in enumerate(moves):
            if mv[1] < 0:
                assert start is None
                start = i
            elif mv[0] < 0:
                assert i - start <= 65
                start = None
        assert start is None
        carry_out(c, moves)
        old = [list(t) for t in m.tokens]
        m.tokens = [old[p] for p in parents]
        m.check()


def test_paged_plan_refuses_and_changes_nothing(lib):
    c = small_cache(4, 4, cap=192)
    m = Model(c)
    m.append(0, 100)
    m.append(1, 70)
    before = books(c)
    for slots, parents, lengths in (([4], [0], [0]), ([-1], [0], [0]), ([2], [4], [0]), ([2], [-1], [0]), ([2], [0], [101]),
                                    ([2], [0], [-2]), ([2, 2], [0, 1], [10, 10])):
        assert plan(lib, c, slots, parents, lengths)[0] == -1
        assert books(c) == before
    assert plan(lib, c, [2, 3], [0, 0], [100, 100])[0] == -3                     # two copies of the last page, none free
    assert books(c) == before and lib.nsa_last_error_string()
    m.check()
    rc, moves = plan(lib, c, [2, 3], [0, 0], [64, 64])                           # whole pages need none
    carry_out(c, moves)
    m.tokens[2] = m.tokens[3] = m.tokens[0][:64]
    m.check()
    rc, moves = plan(lib, c, [1, 2, 3], [0, 0, 0], [100, 100, 0])                # slot 1's pages become the copies
    assert rc == 0
    carry_out(c, moves)
    m.tokens[1] = m.tokens[2] = m.tokens[0]
    m.tokens[3] = []
    m.check()
    assert plan(lib, c, [], [], [])[0] == 0


def test_paged_compaction_plan(lib):
    c = small_cache(4, 20)
    m = Model(c)
    for b in range(4):
        m.append(b, 130 + b)
    carry_out(c, plan(lib, c, [3], [2], [128])[1])
    m.tokens[3] = m.tokens[2][:128]
    for b in (0, 1):
        c.release(b)
        m.tokens[b] = []
    m.check()
    pairs, n, used = (ctypes.c_int32 * (2 * c.num_pages))(), ctypes.c_int32(), ctypes.c_int32()
    args = (c._table, c._lens, c._held, c._refs, c._free.ids, ctypes.byref(c._free.n), c.batch, c.max_pages, c.num_pages,
            pairs, ctypes.byref(n), ctypes.byref(used))
    assert lib.nsa_paged_cache_compact_plan(*args) == 0
    assert used.value == 3 and n.value > 0
    for i in range(n.value):
        src, dst = pairs[2 * i], pairs[2 * i + 1]
        assert src > 3 >= dst
        c.k_pool[dst], c.v_pool_t[dst] = c.k_pool[src], c.v_pool_t[src]
        c.block_table[c.block_table == src] = dst
    m.check()
    assert [c._free[-1 - i] for i in range(3)] == [4, 5, 6]                      # the lowest free page is handed out first
    assert lib.nsa_paged_cache_compact_plan(*args) == 0 and n.value == 0 and used.value == 3


def test_paged_move_argument_errors_do_not_launch(lib):
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    names = ["k", "v", "table", "ck", "cv", "lens", "moves", "n", "batch", "max_pages", "num_pages", "hkv", "dk", "dv",
             "nc_cap", "block", "stride", "dtype", "stream"]
    moves = lambda *a: (ctypes.c_int32 * 40)(*a)                                        # noqa: E731
    good = dict(k=p, v=p, table=p, ck=p, cv=p, lens=p, moves=moves(0, 1, 70, 1, 2), n=1, batch=2, max_pages=4, num_pages=8,
                hkv=2, dk=64, dv=64, nc_cap=64, block=32, stride=16, dtype=0, stream=None)

    def call(**kw):
        return lib.nsa_paged_cache_move(*[dict(good, **kw)[n] for n in names])

    for bad in (dict(k=None), dict(v=None), dict(table=None), dict(ck=None), dict(cv=None), dict(lens=None), dict(moves=None),
                dict(n=-1), dict(batch=0), dict(max_pages=0), dict(num_pages=0), dict(hkv=0), dict(nc_cap=60), dict(block=0),
                dict(stride=0), dict(dtype=9), dict(k=p + 8), dict(ck=p + 4),
                dict(moves=moves(2, 1, 70, 1, 2)), dict(moves=moves(0, 2, 70, 1, 2)), dict(moves=moves(0, 1, 257, 1, 2)),
                dict(moves=moves(0, 1, -1, 1, 2)), dict(moves=moves(0, 1, 70, 8, 2)), dict(moves=moves(0, 1, 70, 1, -1)),
                dict(moves=moves(-1, 1, 70, 1, 2)), dict(moves=moves(-1, -1, 70, 1, 2)),
                dict(moves=moves(0, -1, 70, 1, 2, 1, -1, 70, 1, 2), n=2)):
        assert call(**bad) == -1, bad
    # the register has to be read again, and within a launch
    assert call(moves=moves(0, -1, 70, 1, 2)) == -1
    assert call(moves=moves(0, 1, 70, 1, 2, 1, -1, 70, 1, 2), n=2) == -1
    long = (ctypes.c_int32 * 500)(*([0, -1, 64, 0, 0] + [0, 1, 64, 0, 0] * 79 + [-1, 1, 64, 0, 0]))
    assert call(moves=long, n=81) == -1
    assert call(dk=60) == -2 and call(n=0, moves=None) == 0
    comp = [p, p, p, moves(9, 1), 1, 2, 4, 8, 2, 64, 64, 0, None]
    assert lib.nsa_paged_cache_compact_move(*comp) == -1
    comp[3] = moves(3, 0)
    assert lib.nsa_paged_cache_compact_move(*comp) == -1


def test_paged_cache_python_checks():
    c = small_cache(3, 6)
    c._publish([(0, s, p) for s, p in c._grow(0, 10)])
    c._lens[0] = 10
    for call in (lambda: c.fork(3, 1), lambda: c.fork(-1, 1), lambda: c.fork(0, [0, 1]), lambda: c.fork(0, 1, length=11),
                 lambda: c.fork(0, 1, length=-1), lambda: c.reorder([0, 1]), lambda: c.reorder([0, 1, 3]),
                 lambda: c.reorder([0, 1, -1]), lambda: c.truncate(0, 11), lambda: c.truncate(3, 0), lambda: c.truncate(0, -1)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: c.fork(0, 1), lambda: c.reorder([0, 0, 0]), lambda: c.truncate(0, 5), lambda: c.compact()):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    c.fork(0, [])                                                                # nothing to do
    assert c._lens[0] == 10 and c.free_pages == 5
    with pytest.raises(IndexError):
        c._free[5]
    c.release(-3)                                                                # slots count from the end, as lists do
    assert c.free_pages == 6 and c._lens[0] == 0 and list(c._refs) == [0] * 7
    for b in (3, -4):
        with pytest.raises(IndexError):
            c.release(b)


def test_paged_books_that_are_not_in_order_are_refused(lib):
    """page ids outside the pool, in the table or in the free list, and counts that cannot be: refused, nothing changed"""
    for spoil in range(6):
        c = small_cache(3, 6)
        m = Model(c)
        m.append(0, 100)
        if spoil == 0:
            c._table[1] = 7
        elif spoil == 1:
            c._table[0] = 0
        elif spoil == 2:
            c._held[0] = 6
        elif spoil == 3:
            c._lens[0] = 129
        elif spoil == 4:
            c._free.n.value = 9
        else:
            c._free[-1] = 7
        before = books(c) if spoil != 4 else list(c._refs)
        assert plan(lib, c, [1, 2], [0, 0], [70, 70])[0] == -1
        if spoil != 5:
            assert plan(lib, c, [0], [0], [0])[0] == -1
        if spoil not in (4, 5):
            n = (ctypes.c_int32 * 20)()
            assert lib.nsa_paged_cache_compact_plan(*c._books(), n, ctypes.byref(ctypes.c_int32()),
                                                    ctypes.byref(ctypes.c_int32())) == -1
        assert lib.nsa_paged_cache_grow(*c._books(), 0 if spoil < 4 else 1, 3) == -1
        assert before == (books(c) if spoil != 4 else list(c._refs))
    c = small_cache(2, 6)
    for slot, pages, rc in ((2, 1, -1), (-1, 1, -1), (0, 6, -1), (0, -1, -1), (0, 5, 0), (1, 2, -3), (0, 3, 0)):
        assert lib.nsa_paged_cache_grow(*c._books(), slot, pages) == rc
    assert c._held[0] == 5 and c._held[1] == 0 and c.free_pages == 1


def test_a_copy_of_a_cache_has_books_of_its_own():
    import copy
    c = small_cache(2, 6)
    Model(c).append(0, 70)
    d = copy.deepcopy(c)
    d.release(0)
    assert d.free_pages == 6 and c.free_pages == 4 and c._lens[0] == 70
    Model(d).append(1, 30)
    assert c._held[1] == 0 and d._held[1] == 1


def uneven_full_pool(shared=False):
    """4 pages: slot 0 holds one of them, slot 2 the other three (compression blocks of 64: fill() of fewer tokens runs on
    the CPU)."""
    from nsa_amd.decode import NSAPagedDecodeCache
    c = NSAPagedDecodeCache(3, 4, 192, 1, 8, 8, block=64, dtype=torch.float32, device="cpu")
    c.fill(torch.ones(30, 1, 8), torch.ones(30, 1, 8), seq=0)
    c._publish([(2, s, p) for s, p in c._grow(2, 190)])
    c._lens[2] = 190
    c.ctx_lens[2] = 190
    c._shares = shared
    return c


@pytest.mark.parametrize("shared", [False, True])
def test_fill_takes_the_pages_of_every_slot_it_refills(shared):
    """a full pool whose pages sit in the last slot: all slots are refilled, and both sides of the books agree"""
    c = uneven_full_pool(shared)
    k, v = torch.randn(3, 60, 1, 8), torch.randn(3, 60, 1, 8)
    c.fill(k, v)
    assert list(c._lens) == c.ctx_lens.tolist() == [60] * 3 and list(c._held) == [1] * 3 and c.free_pages == 1
    assert c.block_table.flatten().tolist() == list(c._table)
    pages = [c._pages_of(b)[0] for b in range(3)]
    assert len(set(pages)) == 3 and 0 not in pages and sorted(c._refs) == [0, 0, 1, 1, 1]
    for b, p in enumerate(pages):
        assert torch.equal(c.k_pool[p, :60], k[b]) and torch.equal(c.v_pool_t[p, :, :, :60], v[b].permute(1, 2, 0))
    assert (c.k_pool[0] == 0).all()
    c.fill(k[:, :0], v[:, :0])
    assert c.free_pages == 4 and (c.block_table == 0).all() and (c.ctx_lens == 0).all()


def test_fill_that_does_not_fit_changes_nothing():
    c = uneven_full_pool()
    before = books(c), c.block_table.clone(), c.ctx_lens.clone()
    for T, what in ((65, "exhausted"), (193, "exhausted")):
        with pytest.raises(RuntimeError, match=what):
            c.fill(torch.zeros(3, T, 1, 8), torch.zeros(3, T, 1, 8))
    assert before[0] == books(c) and torch.equal(before[1], c.block_table) and torch.equal(before[2], c.ctx_lens)


def test_a_pickled_cache_comes_back_with_its_books(tmp_path):
    import pickle
    c = small_cache(3, 9)
    m = Model(c)
    m.append(0, 130)
    carry_out(c, plan_of(c, [1], [0], [100]))
    m.tokens[1] = m.tokens[0][:100]
    c.extra = "kept"
    torch.save(c, tmp_path / "cache.pt")
    for d in (pickle.loads(pickle.dumps(c)), torch.load(tmp_path / "cache.pt", weights_only=False)):
        assert books(d) == books(c) and d.extra == "kept" and type(d._table) is type(c._table)
        n = Model(d)
        n.tokens, n.next = [list(t) for t in m.tokens], m.next
        n.check()
        n.append(2, 70)
        d.release(0)
        n.tokens[0] = []
        n.check()
        m.check()


def plan_of(c, slots, parents, lengths):
    moves, n = c._plan(slots, parents, lengths)
    c._shares = True
    return [tuple(moves[5 * i:5 * i + 5]) for i in range(n)]


def test_dense_decode_refuses_results_on_top_of_its_operands(lib):
    """made-up addresses, far apart but for the pair under test: every call is refused before a launch"""
    names = ["q", "k", "v", "table", "max_pages", "num_pages", "lens", "out", "lse", "batch", "hq", "hkv", "dk", "dv", "cap",
             "window", "scale", "dtype", "ws", "ws_bytes", "stream"]
    B, hq, hkv, dk, dv, pages, width = 2, 16, 2, 64, 64, 8, 64
    gap = 1 << 32
    at = {n: (i + 1) * gap for i, n in enumerate(["q", "k", "v", "table", "lens", "out", "lse", "ws"])}
    need = lib.nsa_dense_decode_workspace_bytes(B, hq, hkv, dk, dv, 64 * width, 0, 0)
    size = dict(q=B * hq * dk * 2, k=pages * 64 * hkv * dk * 2, v=pages * 64 * hkv * dv * 2, table=B * width * 4, lens=B * 4,
                out=B * hq * dv * 2, lse=B * hq * 4, ws=need)
    good = dict(at, max_pages=width, num_pages=pages, batch=B, hq=hq, hkv=hkv, dk=dk, dv=dv, cap=0, window=0, scale=0.1,
                dtype=0, ws_bytes=need, stream=None)

    def refused(**kw):
        assert lib.nsa_dense_decode_step(*[dict(good, **kw)[n] for n in names]) == -1, kw
        return b"overlap" in lib.nsa_last_error_string()

    for result in ("out", "lse", "ws"):
        for other in at:
            if other == result:
                continue
            for where in (at[other], at[other] + (size[other] - 1) // 16 * 16, at[other] - (size[result] - 1) // 16 * 16):
                assert refused(**{result: where}), (result, other, where - at[other])
    # a contiguous cache reaches over the whole capacity
    last = at["k"] + B * 64 * width * hkv * dk * 2 - 16
    assert refused(table=None, cap=64 * width, max_pages=0, num_pages=0, out=last)
    # its type decides how far an operand reaches
    assert refused(dtype=1, ws_bytes=1 << 31, out=at["q"] + B * hq * dk * 2)


def test_rope_axes_takes_the_position_type_with_the_axes(lib):
    """refused before a launch: no axes beside the flag, five of them, an axis they do not have, 8-byte positions off by 4"""
    buf = (ctypes.c_char * 4096)()
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 16
    pairs = (ctypes.c_int32 * 128)(0, 1, 2)

    def call(axes, pos=p):
        return lib.nsa_qkv_rope_axes(p, p, p, p, p, p, pos, axes, pairs, 4, 416, 0, 256, 320, 384, 4, 1, 64, 64, 0, 32, 0, 0,
                                     0, None)

    for axes in (256, 256 + 5, 256 + 2, 512 + 3, 3 - 256):
        assert call(axes) == -1
    assert call(256 + 3, p + 4) == -1 and b"aligned to their type" in lib.nsa_last_error_string()
    assert call(3, p + 2) == -1 and b"aligned to their type" in lib.nsa_last_error_string()
