"""GPU tests of the split / rotary step with positions on several axes, forward and backward, against float64.

Bound of the error (u = eps / 2 of the tensors' type, f = 2^-24): the angle reaches the sine in turns with an error of at
most 2^-26 (half a step of fp32 below one half), 2^-23.3 rad, the sine and cosine add at most 4 steps: together below
2^-21 each.  A rotated value is x0 c - x1 s in fp32, so it is off by at most (|x0| + |x1|) (2^-21 + 3 f) and is rounded
once: |y - exact| <= u |exact| + (|x0| + |x1|) 2^-20.  Below the smallest normal number N the steps of the type no longer
shrink with the value: they are eps N there (2^-24 in float16), so the rounding is off by up to u N whatever the value, and
the bound of the rounding is u max(|exact|, N).  Everything that is not rotated has to come through bit for bit."""
import pytest
import torch

from tests.util import randn

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layout(hq, hkv, dk, dv, gap=0, gates=True):
    at = [0, hq * dk + gap, hq * dk + hkv * dk + gap, hq * dk + hkv * (dk + dv) + gap]
    return tuple(at), (at[3] + (3 * hq if gates else 0) + 7) // 8 * 8


def rotated(x, positions, pair_axis, inv_freq, off, interleaved, sign=1.0):
    """x [n, H, dk] on the CPU -> float64 rotated, and the bound without the final rounding."""
    pairs = len(pair_axis)
    x = x.double()
    ang = positions.cpu().double()[list(pair_axis)].t() * inv_freq.cpu().double()
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None] * sign
    first = torch.tensor([off + (2 * i if interleaved else i) for i in range(pairs)])
    second = first + (1 if interleaved else pairs)
    a, b = x[..., first], x[..., second]
    y, slack = x.clone(), torch.zeros_like(x)
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    slack[..., first] = slack[..., second] = (a.abs() + b.abs()) * 2.0 ** -20
    return y, slack


def close(got, ref, slack):
    got = got.detach()
    u = torch.finfo(got.dtype).eps / 2
    still = slack == 0
    got = got.cpu()
    assert torch.equal(got[still].double(), ref[still])            # not rotated, or both channels 0
    rounding = u * ref.abs().clamp(min=torch.finfo(got.dtype).smallest_normal)
    assert bool(((got.double() - ref).abs() <= rounding + slack).all()), \
        float(((got.double() - ref).abs() - rounding - slack).max())


def far_positions(axes, n, seed, top=40000):
    return torch.randint(-5, top, (axes, n), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


def freqs(pairs, theta=10000.0):
    return (1.0 / theta ** (torch.arange(pairs, dtype=torch.float32) / pairs)).to(DEV)


CASES = [
    # hq, hkv, dk, dv, rope_off, rope_dim, axes
    (64, 4, 192, 128, 128, 64, 3),
    (4, 1, 64, 64, 0, 64, 3),
    (12, 4, 128, 128, 0, 128, 2),
    (1, 1, 32, 32, 16, 16, 1),
    (6, 2, 64, 32, 8, 48, 4),
    (2, 1, 256, 8, 0, 256, 3),
    (1, 1, 16, 8, 0, 16, 2),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_split_and_pack(case, dtype, interleaved):
    from nsa_amd import ops
    hq, hkv, dk, dv, off, dim, axes = case
    g = torch.Generator().manual_seed(1)
    pair_axis = [int(a) for a in torch.randint(0, axes, (dim // 2,), generator=g)]
    inv = freqs(dim // 2)
    for n in (1, 2, 7, 63, 300):
        at, ld = layout(hq, hkv, dk, dv)
        kw = dict(inv_freq=inv, positions=far_positions(axes, n, n).to(DEV), rope_off=off, rope_dim=dim,
                  interleaved=interleaved, pair_axis=pair_axis)
        packed = randn(n, ld, seed=3, dtype=dtype)
        q, k, v, gates = ops.qkv_rope_split(packed.to(DEV), hq, hkv, dk, dv, at, **kw)
        for got, lo, h in ((q, at[0], hq), (k, at[1], hkv)):
            x = packed[:, lo:lo + h * dk].reshape(n, h, dk)
            close(got, *rotated(x, kw["positions"], pair_axis, inv, off, interleaved))
        assert torch.equal(v.cpu().view(n, -1), packed[:, at[2]:at[3]])
        assert torch.equal(gates.cpu().view(n, -1), packed[:, at[3]:at[3] + 3 * hq])
        grads = [randn(*t.shape, seed=4 + i, dtype=dtype) for i, t in enumerate((q, k, v, gates))]
        d = ops.qkv_rope_pack(*[t.to(DEV) for t in grads], ld, at, **kw).cpu()
        for i, (lo, h) in enumerate(((at[0], hq), (at[1], hkv))):
            close(d[:, lo:lo + h * dk].reshape(n, h, dk),
                  *rotated(grads[i], kw["positions"], pair_axis, inv, off, interleaved, -1.0))
        assert torch.equal(d[:, at[2]:at[3]], grads[2].view(n, -1))
        assert torch.equal(d[:, at[3]:at[3] + 3 * hq], grads[3].view(n, -1))
        assert (d[:, at[3] + 3 * hq:] == 0).all()


@pytest.mark.parametrize("n", [5003, 20011])
def test_many_rows(n):
    """beyond the size from which a thread takes several items; an odd number of rows"""
    from nsa_amd import ops
    hq, hkv, dk, dv, dim, dtype = 16, 2, 64, 64, 32, torch.bfloat16
    at, ld = layout(hq, hkv, dk, dv)
    pair_axis, inv = [i % 3 for i in range(16)], freqs(16)
    pos = far_positions(3, n, 8).to(DEV)
    packed = randn(n, ld, seed=9, dtype=dtype)
    kw = dict(inv_freq=inv, positions=pos, rope_off=32, rope_dim=dim, interleaved=False, pair_axis=pair_axis)
    q, k, v, gates = ops.qkv_rope_split(packed.to(DEV), hq, hkv, dk, dv, at, **kw)
    close(q, *rotated(packed[:, :at[1]].reshape(n, hq, dk), pos, pair_axis, inv, 32, False))
    close(k, *rotated(packed[:, at[1]:at[2]].reshape(n, hkv, dk), pos, pair_axis, inv, 32, False))
    assert torch.equal(v.cpu().view(n, -1), packed[:, at[2]:at[3]])
    assert torch.equal(gates.cpu().view(n, -1), packed[:, at[3]:at[3] + 3 * hq])
    d = ops.qkv_rope_pack(q, k, v, gates, ld, at, **kw).cpu()
    close(d[:, :at[1]].reshape(n, hq, dk), *rotated(q.cpu(), pos, pair_axis, inv, 32, False, -1.0))
    assert (d[:, at[3] + 3 * hq:] == 0).all()


@pytest.mark.parametrize("seed", range(24))
def test_random_layouts(seed):
    """heads, head dims, rotary ranges, gaps, gate alignment, axes, types and row counts drawn together"""
    import random
    from nsa_amd import ops
    g = random.Random(seed)
    dtype = g.choice([torch.bfloat16, torch.float16, torch.float32])
    interleaved = g.random() < 0.5
    hq, hkv = g.randint(1, 20), g.randint(1, 6)
    dk, dv = 8 * g.randint(2, 32), 8 * g.randint(1, 20)
    unit = 8 if interleaved else 16
    dim = unit * g.randint(1, dk // unit)
    off = 8 * g.randint(0, (dk - dim) // 8)
    axes, n = g.randint(1, 4), g.choice([1, 3, 17, 64, 129, 1500])
    gap = 8 * g.choice([0, 0, 1, 3])
    with_gates = g.random() < 0.8
    at = [0, hq * dk + gap, hq * dk + hkv * dk + gap, hq * dk + hkv * (dk + dv) + gap + g.choice([0, 0, 3])]
    ld = (at[3] + 3 * hq + 7) // 8 * 8 + 8 * g.choice([0, 2])
    pair_axis = [g.randrange(axes) for _ in range(dim // 2)]
    inv = freqs(dim // 2)
    pos = far_positions(axes, n, seed).to(DEV)
    packed = randn(n, ld, seed=seed, dtype=dtype)
    kw = dict(inv_freq=inv, positions=pos, rope_off=off, rope_dim=dim, interleaved=interleaved, pair_axis=pair_axis)
    q, k, v, gates = ops.qkv_rope_split(packed.to(DEV), hq, hkv, dk, dv, tuple(at), with_gates=with_gates, **kw)
    close(q, *rotated(packed[:, :hq * dk].reshape(n, hq, dk), pos, pair_axis, inv, off, interleaved))
    close(k, *rotated(packed[:, at[1]:at[1] + hkv * dk].reshape(n, hkv, dk), pos, pair_axis, inv, off, interleaved))
    assert torch.equal(v.cpu().view(n, -1), packed[:, at[2]:at[2] + hkv * dv])
    assert (gates is None) != with_gates
    if with_gates:
        assert torch.equal(gates.cpu().view(n, -1), packed[:, at[3]:at[3] + 3 * hq])
    d = ops.qkv_rope_pack(q, k, v, gates, ld, tuple(at), **kw).cpu()
    close(d[:, :hq * dk].reshape(n, hq, dk), *rotated(q.cpu(), pos, pair_axis, inv, off, interleaved, -1.0))
    close(d[:, at[1]:at[1] + hkv * dk].reshape(n, hkv, dk), *rotated(k.cpu(), pos, pair_axis, inv, off, interleaved, -1.0))
    assert torch.equal(d[:, at[2]:at[2] + hkv * dv], v.cpu().view(n, -1))
    rest = torch.ones(ld, dtype=torch.bool)
    for lo, w in ((0, hq * dk), (at[1], hkv * dk), (at[2], hkv * dv), (at[3], 3 * hq if with_gates else 0)):
        rest[lo:lo + w] = False
    assert (d[:, rest] == 0).all()
    if with_gates:
        assert torch.equal(d[:, at[3]:at[3] + 3 * hq], gates.cpu().view(n, -1))


def test_positions_at_the_ends_of_their_range():
    from nsa_amd import ops
    hq, hkv, dk, dv, dim = 2, 1, 64, 64, 64
    at, ld = layout(hq, hkv, dk, dv)
    pos = torch.tensor([[0, 2 ** 31 - 1, -2 ** 31, 1_000_003, -7], [1, 2 ** 30 + 1, 5, -2 ** 31 + 1, 99]], dtype=torch.int32)
    pair_axis, inv = [i % 2 for i in range(32)], freqs(32)
    packed = randn(5, ld, seed=10)
    q = ops.qkv_rope_split(packed.to(DEV), hq, hkv, dk, dv, at, inv_freq=inv, positions=pos.to(DEV), rope_off=0,
                           rope_dim=dim, pair_axis=pair_axis)[0]
    close(q, *rotated(packed[:, :at[1]].reshape(5, hq, dk), pos, pair_axis, inv, 0, False))


def test_gaps_strides_and_position_types():
    """ranges in another order with a gap between them, rows of a wider tensor, positions as int64 and transposed"""
    from nsa_amd import ops
    hq, hkv, dk, dv, dim, n, dtype = 4, 2, 64, 32, 32, 77, torch.bfloat16
    at = (hkv * dk + 16, 0, hkv * dk + 16 + hq * dk, hkv * (dk + dv) + 16 + hq * dk + 5)      # k, gap, q, v, gap, gates
    ld = (at[3] + 3 * hq + 7) // 8 * 8 + 8
    pair_axis, inv = [0] * 4 + [1] * 6 + [2] * 6, freqs(16)
    pos = far_positions(3, n, 12).to(DEV)
    wide = randn(n, 2 * ld, seed=13, dtype=dtype).to(DEV)
    kw = dict(inv_freq=inv, rope_off=16, rope_dim=dim, interleaved=True, pair_axis=pair_axis)
    q, k, v, gates = ops.qkv_rope_split(wide[:, ld:], hq, hkv, dk, dv, at, positions=pos.long().t().contiguous().t(), **kw)
    packed = wide[:, ld:].cpu()
    close(q, *rotated(packed[:, at[0]:at[0] + hq * dk].reshape(n, hq, dk), pos, pair_axis, inv, 16, True))
    close(k, *rotated(packed[:, :hkv * dk].reshape(n, hkv, dk), pos, pair_axis, inv, 16, True))
    assert torch.equal(gates.cpu().view(n, -1), packed[:, at[3]:at[3] + 3 * hq])
    q2, k2, v2, g2 = ops.qkv_rope_split(wide[:, ld:], hq, hkv, dk, dv, at, positions=pos, with_gates=False, **kw)
    assert g2 is None and torch.equal(q2, q) and torch.equal(k2, k) and torch.equal(v2, v)
    d = ops.qkv_rope_pack(q, k, v, gates, ld, at, positions=pos, **kw).cpu()
    for lo, hi in ((hkv * dk, at[0]), (at[2] + hkv * dv, at[3]), (at[3] + 3 * hq, ld)):
        assert (d[:, lo:hi] == 0).all()
    close(d[:, at[0]:at[0] + hq * dk].reshape(n, hq, dk), *rotated(q.cpu(), pos, pair_axis, inv, 16, True, -1.0))
    empty = ops.qkv_rope_split(wide[:0, ld:], hq, hkv, dk, dv, at, positions=pos[:, :0], **kw)
    assert [t.shape[0] for t in empty] == [0, 0, 0, 0]


def test_offsets_beyond_32_bits():
    """a packed tensor of more than 2^31 elements: its first and last rows"""
    from nsa_amd import ops
    hq, hkv, dk, dv, dim, dtype = 64, 4, 192, 128, 64, torch.bfloat16
    at, ld = layout(hq, hkv, dk, dv)
    n = 2 ** 31 // ld + 1000
    pair_axis, inv = [0] * 8 + [1] * 12 + [2] * 12, freqs(32)
    pos = far_positions(3, n, 14).to(DEV)
    packed = torch.empty(n, ld, dtype=dtype, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(2))
    kw = dict(inv_freq=inv, positions=pos, rope_off=128, rope_dim=dim, pair_axis=pair_axis)
    q, k, v, gates = ops.qkv_rope_split(packed, hq, hkv, dk, dv, at, **kw)
    d = ops.qkv_rope_pack(q, k, v, gates, ld, at, **kw)
    for rows in (slice(0, 50), slice(n - 50, n)):
        x = packed[rows].cpu()
        close(q[rows], *rotated(x[:, :at[1]].reshape(50, hq, dk), pos[:, rows], pair_axis, inv, 128, False))
        close(k[rows], *rotated(x[:, at[1]:at[2]].reshape(50, hkv, dk), pos[:, rows], pair_axis, inv, 128, False))
        assert torch.equal(v[rows].cpu().view(50, -1), x[:, at[2]:at[3]])
        close(d[rows, :at[1]].reshape(50, hq, dk), *rotated(q[rows].cpu(), pos[:, rows], pair_axis, inv, 128, False, -1.0))


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_the_formula_and_differences(interleaved):
    from nsa_amd.autograd import QkvRopeFn
    hq, hkv, dk, dv, dim, n = 4, 2, 64, 32, 32, 9
    at, ld = layout(hq, hkv, dk, dv)
    pair_axis, inv = [i % 3 for i in range(16)], freqs(16)
    pos = far_positions(3, n, 15, top=300).to(DEV)
    x = randn(n, ld, seed=16).to(DEV).requires_grad_(True)
    args = (hq, hkv, dk, dv, at, inv, pos, None, 32, dim, interleaved, True, pair_axis)
    outs = QkvRopeFn.apply(x, *args)
    w = [randn(*t.shape, seed=17 + i).to(DEV) for i, t in enumerate(outs)]
    sum((t * u).sum() for t, u in zip(outs, w)).backward()
    grad = x.grad.cpu()
    close(grad[:, :at[1]].reshape(n, hq, dk), *rotated(w[0].cpu(), pos, pair_axis, inv, 32, interleaved, -1.0))
    close(grad[:, at[1]:at[2]].reshape(n, hkv, dk), *rotated(w[1].cpu(), pos, pair_axis, inv, 32, interleaved, -1.0))
    # the step is linear: a difference of any width equals the slope, to the rounding of both sides
    for seed in range(3):
        step = randn(n, ld, seed=30 + seed).to(DEV)
        with torch.no_grad():
            up, down = QkvRopeFn.apply(x + step, *args), QkvRopeFn.apply(x - step, *args)
            slope = sum(((a.double() - b.double()) / 2 * u.double()).sum() for a, b, u in zip(up, down, w))
        want = (grad.double() * step.cpu().double()).sum()
        size = sum((u.double().abs() * (x.abs().max() + step.abs().max()).double()).sum() for u in w)
        assert abs(float(slope.detach().cpu() - want.detach())) <= float(size.detach()) * 2.0 ** -18
    # some outputs unused
    x.grad = None
    QkvRopeFn.apply(x, *args)[1].sum().backward()
    assert (x.grad[:, :at[1]] == 0).all() and (x.grad[:, at[2]:] == 0).all() and x.grad[:, at[1]:at[2]].abs().max() > 0


def test_positions_changed_before_the_backward_are_noticed():
    from nsa_amd.autograd import QkvRopeFn
    at, ld = layout(2, 1, 32, 32)
    pos = far_positions(2, 4, 18).to(DEV)
    x = randn(4, ld, seed=19).to(DEV).requires_grad_(True)
    out = QkvRopeFn.apply(x, 2, 1, 32, 32, at, freqs(16), pos, None, 0, 32, False, True, [0, 1] * 8)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        out[0].sum().backward()


def test_equal_axes_are_the_single_axis_rotation():
    """the same place on every axis: the kernel of one axis, whose angles are fp32 products"""
    from nsa_amd import ops
    hq, hkv, dk, dv, dim, n = 8, 2, 64, 64, 64, 200
    at, ld = layout(hq, hkv, dk, dv)
    packed = randn(n, ld, seed=20).to(DEV)
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    one = ops.qkv_rope_split(packed, hq, hkv, dk, dv, at, freqs(32), pos, None, 0, dim)
    many = ops.qkv_rope_split(packed, hq, hkv, dk, dv, at, freqs(32), pos.expand(3, n), None, 0, dim,
                              pair_axis=[i % 3 for i in range(32)])
    # |angle| <= 200: its product is off by at most 200 * 2^-24 rad; inputs below 5
    for a, b in zip(one, many):
        assert float((a - b).abs().max()) <= 2 * 5 * (200 * 2.0 ** -24 + 2.0 ** -20)


def test_captured_calls_and_other_streams():
    from nsa_amd import ops
    hq, hkv, dk, dv, dim, n, dtype = 8, 2, 64, 64, 32, 33, torch.bfloat16
    at, ld = layout(hq, hkv, dk, dv)
    kw = dict(inv_freq=freqs(16), rope_off=32, rope_dim=dim, pair_axis=[0] * 4 + [1] * 6 + [2] * 6)
    x = torch.zeros(n, ld, dtype=dtype, device=DEV)
    pos = torch.zeros(3, n, dtype=torch.int32, device=DEV)
    run = lambda: ops.qkv_rope_split(x, hq, hkv, dk, dv, at, positions=pos, **kw)     # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
        back = ops.qkv_rope_pack(*outs, ld, at, positions=pos, **kw)
    side = torch.cuda.Stream()
    for s in range(5):
        x.copy_(randn(n, ld, seed=40 + s, dtype=dtype))
        pos.copy_(far_positions(3, n, 50 + s))
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = run()
            eager_back = ops.qkv_rope_pack(*eager, ld, at, positions=pos, **kw)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)) and torch.equal(back, eager_back), s


# ------------------------------------------------------------------------------------------------------- the layer

def make_layer(rope_axes, seed=0, **kw):
    from nsa_amd.layer import NSAAttentionLayer
    torch.manual_seed(seed)
    return NSAAttentionLayer(256, 8, 2, 64, rope_dim=32, compressor_mode="mean", gate_activation="sigmoid",
                             selected_block_count=4, sliding_window=64, rope_axes=rope_axes, device=DEV,
                             dtype=torch.bfloat16, **kw)


def test_layer_with_equal_axes_is_the_layer_with_one():
    B, T = 2, 150
    x = randn(B, T, 256, seed=60, scale=0.5, dtype=torch.bfloat16).to(DEV)
    one, many = make_layer(None), make_layer((4, 6, 6), rope_axes_layout="turns")
    many.load_state_dict(one.state_dict())
    pos = torch.arange(T, device=DEV).expand(3, B, T)
    with torch.no_grad():
        a, b, c = one(x)[0], many(x)[0], many(x, position_ids=pos)[0]
    assert torch.equal(b, c)
    u = torch.finfo(torch.bfloat16).eps / 2
    # q and k may differ by one rounding; picks of near ties aside, the outputs by a few
    assert float((a - b).abs().float().mean()) <= 4 * u * float(a.abs().float().mean())
    cu = torch.tensor([0, 60, 150], dtype=torch.int32, device=DEV)
    packed = x.reshape(-1, 256)[:150]
    place = torch.cat([torch.arange(60), torch.arange(90)]).to(DEV)
    with torch.no_grad():
        d = many(packed, cu_seqlens=cu, max_seqlen=90)[0]
        e = many(packed, cu_seqlens=cu, max_seqlen=90, position_ids=place.expand(3, 150))[0]
    assert torch.equal(d, e)


def test_layer_gradients_reach_the_projections_through_the_rotation():
    """d_out -> dq of the attention -> inverse rotation -> q_proj: the same layer with the rotation in float64 torch, run
    over the q, k, v gradients that the attention hands back"""
    from nsa_amd import ops
    from nsa_amd.autograd import QkvRopeFn
    T = 130
    layer = make_layer((4, 6, 6))
    x = randn(1, T, 256, seed=61, scale=0.5, dtype=torch.bfloat16).to(DEV)
    pos = far_positions(3, T, 62, top=2000).to(DEV)
    seen = {}
    split, pack = ops.qkv_rope_split, ops.qkv_rope_pack

    def spy(*a, **kw):
        seen["grads"] = [t.detach().clone() for t in a[:4]]
        seen["packed"] = pack(*a, **kw)
        return seen["packed"]

    ops.qkv_rope_pack = spy
    try:
        out, _ = layer(x, position_ids=pos.view(3, 1, T))
        out.float().square().sum().backward()
    finally:
        ops.qkv_rope_pack = pack
    d = seen["packed"].cpu()
    dq, dk = seen["grads"][0].cpu(), seen["grads"][1].cpu()
    at = layer.offsets
    close(d[:, at[0]:at[1]].reshape(T, 8, 64), *rotated(dq, pos, layer.pair_axis, layer.inv_freq, 32, False, -1.0))
    close(d[:, at[1]:at[2]].reshape(T, 2, 64), *rotated(dk, pos, layer.pair_axis, layer.inv_freq, 32, False, -1.0))
    want = d[:, at[1]:at[2]].double().t() @ x[0].cpu().double()
    got = layer.k_proj.weight.grad.cpu().double()
    u = torch.finfo(torch.bfloat16).eps / 2
    size = d[:, at[1]:at[2]].double().abs().t() @ x[0].cpu().double().abs()
    assert ((got - want).abs() <= u * want.abs() + size * (T + 8) * 2.0 ** -24).all()
    for name, p in layer.named_parameters():
        if "compressor" not in name:                 # the mean compressor does not use its weights
            assert p.grad is not None and torch.isfinite(p.grad).all(), name


def test_layer_decode_step_takes_the_new_tokens_positions():
    from nsa_amd.decode import NSAPagedDecodeCache
    B, T = 2, 100
    layer = make_layer((4, 6, 6), rope_axes_spectrum="own")
    x = randn(B, T + 1, 256, seed=63, scale=0.5, dtype=torch.bfloat16).to(DEV)
    pos = far_positions(3, B * (T + 1), 64, top=500).view(3, B, T + 1).to(DEV)
    with torch.no_grad():
        rows = layer(x, position_ids=pos)[0][:, -1]
        steps = []
        for last in (pos[:, :, T:], pos[:, :, T]):
            cache = NSAPagedDecodeCache(B, 8, 128, 2, 64, 64, device=DEV)
            layer(x[:, :T], position_ids=pos[:, :, :T], past_key_value=cache)
            steps.append(layer(x[:, T:], position_ids=last, past_key_value=cache)[0][:, 0])
    assert torch.equal(steps[0], steps[1])
    # the decode step and the prefill row round probabilities, branches and the projection separately
    u = torch.finfo(torch.bfloat16).eps / 2
    assert float((steps[0] - rows).abs().float().mean()) <= 8 * u * float(rows.abs().float().mean())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_positions_beyond_32_bits_keep_all_of_theirs(dtype):
    """int64 positions, forward and backward.  The angle is a product of two rounded 64-bit numbers there, in the reference
    too, each off by 2^-52 of itself at most: the bound has |angle| 2^-51 more."""
    from nsa_amd import ops
    from nsa_amd.autograd import QkvRopeFn
    hq, hkv, dk, dv, dim = 4, 2, 64, 64, 64
    at, ld = layout(hq, hkv, dk, dv)
    pos = torch.tensor([[2 ** 31, -2 ** 31 - 1, 2 ** 32 + 5, 7, -2 ** 34 - 99, 3], [0, 2 ** 33 + 2 ** 20 + 1, -1, 2 ** 31 + 12345,
                        2 ** 35 + 17, -2 ** 31]])
    pair_axis, inv = [i % 2 for i in range(32)], freqs(32)
    far = (pos.double().abs().amax(0) * 2.0 ** -51)[:, None, None]
    kw = dict(inv_freq=inv, positions=pos.to(DEV), rope_off=0, rope_dim=dim, pair_axis=pair_axis)

    def check(got, x, sign):
        ref, slack = rotated(x, pos, pair_axis, inv, 0, False, sign)
        x = x.double().abs()
        close(got, ref, slack + (x + x.roll(32, -1)) * far)

    packed = randn(6, ld, seed=17, dtype=dtype)
    q, k, v, gates = ops.qkv_rope_split(packed.to(DEV), hq, hkv, dk, dv, at, **kw)
    check(q, packed[:, :at[1]].reshape(6, hq, dk), 1.0)
    check(k, packed[:, at[1]:at[2]].reshape(6, hkv, dk), 1.0)
    d = ops.qkv_rope_pack(q, k, v, gates, ld, at, **kw).cpu()
    check(d[:, :at[1]].reshape(6, hq, dk), q.cpu(), -1.0)
    x = packed.to(DEV).requires_grad_()
    outs = QkvRopeFn.apply(x, hq, hkv, dk, dv, at, inv, kw["positions"], None, 0, dim, False, True, pair_axis)
    assert torch.equal(outs[0], q)
    torch.autograd.backward(outs, [t.detach() for t in outs])
    assert torch.equal(x.grad.cpu(), d)
    # and those that fit are the same in either type
    near = torch.tensor([[2 ** 31 - 1, -2 ** 31, 5, 0, -9, 77]] * 2)
    both = [ops.qkv_rope_split(packed.to(DEV), hq, hkv, dk, dv, at, **dict(kw, positions=near.to(DEV, t)))[0]
            for t in (torch.int64, torch.int32)]
    assert torch.equal(*both)
