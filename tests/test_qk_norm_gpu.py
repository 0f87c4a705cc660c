"""GPU tests of the norm and rotation of query and key heads (kernels/hip/qk_norm.py) against float64, with bounds counted from
the kernels' roundings."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0**-24  # half a step of fp32
EPS = 1e-5


def _call(*args, **kw):
    from nanonemo_amd.kernels.hip.qk_norm import qk_norm_rope

    return qk_norm_rope(*args, **kw)


def _tables(rows, D):
    angle = torch.outer(torch.arange(rows, dtype=torch.float64), 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    return angle.cos().float().cuda(), angle.sin().float().cuda()


def _inputs(lead, H, KVH, D, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, dq, dk = ((s * torch.randn(*lead, n, D, device="cuda", generator=g)).to(dtype) for n, s in ((H, 2.0), (KVH, 0.5), (H, 1.0), (KVH, 1.0)))
    wq, wk = (1 + 0.3 * torch.randn(D, device="cuda", generator=g) for _ in range(2))
    return q, k, wq, wk, dq, dk


def _float64(x, w, dy, cos, sin, positions, eps=EPS):
    """The output and gradients, and for each the bound of its error but for the last rounding:

    r: a lane adds 16 squares and a team's butterfly up to 4 more steps, all positive: 20 U of the sum, half of that in r, and
    the reciprocal root's own step 2 U, a product and a sum 1 U: 13 U. v = (x r) w: 15 U. y: a product and a sum each, 17 U of
    the two terms; 20 U with the second-order ones.
    g = R^T dy: 2 U of its two terms G = |d1| + |d2| (cos, sin <= 1). w g: 3 U. n = x r: 14 U. m = mean(w g n): 3 + 20 of its terms,
    r and two products: 39 U of their mean M. dx = r (w g - n m): 13 + 2 more: 18 U of G |w| r and 70 U of |n| M r.
    dw: terms 17 U; a thread adds up to 100 of them one by one, 6 butterfly steps, 4 waves, 64 rows and 16 sums: 190 U."""
    x, w, c, s = x.double(), w.double(), cos.double()[positions].unsqueeze(-2), sin.double()[positions].unsqueeze(-2)
    half = x.shape[-1] // 2

    def pair(a, b):
        return torch.cat((a, b), -1)

    r = 1 / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    n = x * r
    v1, v2 = (w * n).split(half, -1)
    y, ybound = pair(v1 * c - v2 * s, v1 * s + v2 * c), pair(*[20 * U * (v1.abs() + v2.abs())] * 2)
    d1, d2 = dy.double().split(half, -1)
    g, G = pair(d1 * c + d2 * s, d2 * c - d1 * s), pair(*[d1.abs() + d2.abs()] * 2)
    dx = r * (w * g - n * (w * g * n).mean(-1, keepdim=True))
    xbound = U * r * (20 * G * w.abs() + 70 * n.abs() * (G * w.abs() * n.abs()).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    return (y, ybound), (dx, xbound), ((g * n).sum(lead), 190 * U * (G * n.abs()).sum(lead))


def _check(got, want, what):
    ref, bound = want
    assert got.shape == ref.shape, what
    err = (got.double() - ref).abs() - torch.finfo(got.dtype).eps / 2 * ref.abs() * 1.01 - bound - torch.finfo(got.dtype).tiny
    assert (err <= 0).all(), (what, err.max().item())


# leading sizes, H, KVH, hd: one token; a decode step; teams with idle lanes (48, 80, 96, 240); heads that leave a unit part empty;
# enough tokens that a team of the backward walks several units.
CASES = [((1,), 1, 1, 16), ((7,), 12, 4, 64), ((2, 5), 5, 3, 48), ((1, 33), 9, 1, 80), ((3, 130), 8, 8, 128), ((77,), 3, 2, 96), ((19,), 2, 2, 240), ((4, 9), 4, 1, 256), ((2, 1024), 12, 4, 64),
         ((9000,), 12, 4, 64), ((3001,), 4, 2, 32)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lead, H, KVH, D", CASES)
def test_matches_float64(lead, H, KVH, D, dtype):
    print(f"\n[case] qk_norm lead={lead} H={H} KVH={KVH} D={D} {dtype}", flush=True)
    q, k, wq, wk, dq, dk = _inputs(lead, H, KVH, D, dtype)
    cos, sin = _tables(max(600, lead[-1]), D)
    positions = torch.randint(0, 600, lead, device="cuda")
    for pos in (None, positions, positions.int()):
        at = torch.arange(lead[-1], device="cuda").expand(lead) if pos is None else positions
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        outs = _call(*leaves, cos, sin, pos)
        gq, gk, gwq, gwk = torch.autograd.grad(outs, leaves, (dq, dk))
        for x, w, dy, y, dx, dw, what in ((q, wq, dq, outs[0], gq, gwq, "q"), (k, wk, dk, outs[1], gk, gwk, "k")):
            for got, want, name in zip((y, dx, dw), _float64(x, w, dy, cos, sin, at), ("y", "dx", "dw")):
                _check(got.detach(), want, (what, name))
            assert y.dtype == dx.dtype == dtype and dw.dtype == torch.float32 and y.is_contiguous()


def test_gradients_match_differences():
    q, k, wq, wk, dq, dk = _inputs((6,), 3, 2, 32, torch.float32, seed=1)
    cos, sin = _tables(10, 32)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(_call(*leaves, cos, sin), leaves, (dq, dk))

    def loss(ins):
        return sum((y.double() * d.double()).sum() for y, d in zip(_call(*ins, cos, sin), (dq, dk))).item()

    h, g = 2.0**-7, torch.Generator(device="cuda").manual_seed(2)
    with torch.no_grad():
        for i, grad in enumerate(grads):
            step = h * torch.sign(torch.randn(grad.shape, device="cuda", generator=g))
            ins = [list(leaves), list(leaves)]
            ins[0][i], ins[1][i] = leaves[i] + step, leaves[i] - step
            want, got = (loss(ins[0]) - loss(ins[1])) / (2 * h), (grad.double() * step.double()).sum().item() / h
            # third derivatives: h^2 / 6 of terms of up to some tens (1 / rms^3 of a vector); rounding: 20 U of 192 outputs of
            # about 1, over h
            assert abs(want - got) <= 1e-2 * max(1.0, grad.double().norm().item()), (i, want, got)


def test_a_position_for_each_row_or_for_each_column():
    q, k, wq, wk, _, _ = _inputs((3, 8), 4, 2, 64, torch.bfloat16)
    cos, sin = _tables(50, 64)
    pos = torch.randint(0, 50, (8,), device="cuda")
    a, b = _call(q, k, wq, wk, cos, sin, pos), _call(q, k, wq, wk, cos, sin, pos.expand(3, 8))
    c = _call(q, k, wq, wk, cos[pos].contiguous(), sin[pos].contiguous())
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))


def test_projections_are_read_in_place_and_other_layouts_copied():
    H, KVH, D, T = 12, 4, 64, 50
    q, k, wq, wk, dq, dk = _inputs((T,), H, KVH, D, torch.bfloat16, seed=3)
    cos, sin = _tables(T, D)

    def run(q, k, dq, dk):
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        outs = _call(*leaves, cos, sin)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, (dq, dk)))

    ref = run(q, k, dq, dk)
    wide = torch.cat([q.view(T, -1), k.view(T, -1), k.view(T, -1)], 1)
    cols = [t.view(T, -1, D) for t in wide.split([H * D, KVH * D, KVH * D], 1)]
    assert all(torch.equal(a, b) for a, b in zip(run(*cols[:2], dq, dk), ref))
    turn = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, dq, dk)]
    odd = [torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape) for t in (q, k, dq, dk)]
    apart = [torch.stack([t, t], -1)[..., 1] for t in (q, k, dq, dk)]
    back = [t.flip(0).contiguous().as_strided(t.shape, t.stride()).flip(0) for t in (q, k, dq, dk)]
    for views in (turn, odd, apart, back):
        assert all(torch.equal(a, b) for a, b in zip(run(*views), ref))
    one = dq[:, :1, :1].expand(T, H, D)
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, one, dk), run(q, k, one.contiguous(), dk)))
    q4, k4 = (t.view(2, T // 2, -1, D) for t in cols[:2])  # a batch of a projection's rows, every other token of it
    a = _call(q4[:, ::2], k4[:, ::2], wq, wk, cos, sin)
    b = _call(q4[:, ::2].contiguous(), k4[:, ::2].contiguous(), wq, wk, cos, sin)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for w in (torch.cat([wq.new_zeros(1), wq])[1:], torch.stack([wq, wq], 1)[:, 0]):
        assert torch.equal(_call(q, k, w, wk, cos, sin)[0], ref[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_positions_out_of_the_tables_and_special_values(dtype):
    print(f"\n[case] qk_norm special values {dtype}", flush=True)
    q, k, wq, wk, dq, dk = _inputs((9,), 3, 2, 64, dtype, seed=4)
    cos, sin = _tables(20, 64)
    pos = torch.tensor([3, 20, 19, -1, 0, 1 << 40, 5, 6, 7], device="cuda")
    good = (pos >= 0) & (pos < 20)
    y = _call(q, k, wq, wk, cos, sin, pos)
    ref = _call(q, k, wq, wk, cos, sin, pos.clamp(0, 19))
    for a, b in zip(y, ref):
        assert a[~good].isnan().all() and torch.equal(a[good], b[good])
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    gq, gk, gwq, gwk = torch.autograd.grad(_call(*leaves, cos, sin, pos), leaves, (dq, dk))
    assert gq[~good].isnan().all() and gk[~good].isnan().all() and gq[good].isfinite().all() and gwq.isnan().all() and gwk.isnan().all()
    with torch.no_grad():  # a NaN or an infinity stays in its vector; a vector of zeros is zeros
        x = q.detach().clone()
        x[1, 1, 5], x[2, 0, 3], x[4, 2] = float("nan"), float("inf"), 0.0
        a, b = _call(x, k, wq, wk, cos, sin)[0], _call(q, k, wq, wk, cos, sin)[0]
        assert a[1, 1].isnan().all() and a[2, 0].isnan().any() and (a[4, 2] == 0).all()
        rest = torch.ones(9, 3, dtype=torch.bool, device="cuda")
        rest[1, 1] = rest[2, 0] = rest[4, 2] = False
        assert torch.equal(a[rest], b[rest])
    x = torch.zeros_like(q).requires_grad_()
    (gx,) = torch.autograd.grad(_call(x, k, wq, wk, cos, sin)[0], x, dq)  # of a vector of zeros: w g / sqrt(eps)
    _check(gx, _float64(x.detach(), wq.detach(), dq, cos, sin, torch.arange(9, device="cuda"))[1], "zeros")


def test_either_output_alone_and_nothing_to_do():
    q, k, wq, wk, dq, dk = _inputs((30,), 4, 2, 64, torch.bfloat16, seed=5)
    cos, sin = _tables(30, 64)
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    both = torch.autograd.grad(_call(*leaves, cos, sin), leaves, (dq, dk))
    only_q = torch.autograd.grad(_call(*leaves, cos, sin)[0], leaves, dq, allow_unused=True)
    only_k = torch.autograd.grad(_call(*leaves, cos, sin)[1], leaves, dk, allow_unused=True)
    assert torch.equal(both[0], only_q[0]) and torch.equal(both[2], only_q[2]) and torch.equal(both[1], only_k[1]) and torch.equal(both[3], only_k[3])
    assert not only_q[1].any() and not only_q[3].any() and not only_k[0].any() and not only_k[2].any()
    empty = [t.detach()[:0].requires_grad_() for t in (q, k)]
    outs = _call(*empty, wq, wk, cos, sin)
    g = torch.autograd.grad(outs, (*empty, wq, wk), [torch.empty_like(t) for t in outs])
    assert [t.shape[0] for t in g] == [0, 0, 64, 64] and not g[2].any() and not g[3].any()


def test_op_and_eager_path_give_the_same_bits_and_the_op_passes_opcheck():
    q, k, wq, wk, dq, dk = _inputs((2, 30), 4, 2, 64, torch.float16, seed=6)
    cos, sin = _tables(40, 64)
    pos = torch.randint(0, 40, (2, 30), device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    outs, op = _call(*leaves, cos, sin, pos), torch.ops.nanonemo.qk_norm_rope(*leaves, cos, sin, pos, EPS)
    assert "QkNormNode" in outs[0].grad_fn.name() and all(torch.equal(a, b) for a, b in zip(outs, op))
    ref = torch.autograd.grad(outs, leaves, (dq, dk))
    assert all(torch.equal(a, b) for a, b in zip(ref, torch.autograd.grad(op, leaves, (dq, dk))))
    torch.library.opcheck(torch.ops.nanonemo.qk_norm_rope, (*leaves, cos, sin, pos, EPS))
    torch.library.opcheck(torch.ops.nanonemo.qk_norm_rope, (*leaves, cos, sin, None, EPS))
    torch.library.opcheck(torch.ops.nanonemo.qk_norm_rope_bwd, (dq, dk, *(t.detach() for t in leaves), cos, sin, pos, EPS))
    f = torch.compile(lambda *ins: [2 * t for t in _call(*ins, cos, sin, pos)], fullgraph=True, backend="aot_eager")
    got = f(*leaves)
    assert all(torch.equal(a, 2 * b) for a, b in zip(got, outs))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, (dq, dk)), torch.autograd.grad([2 * t for t in _call(*leaves, cos, sin, pos)], leaves, (dq, dk))))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(_call(*leaves, cos, sin, pos), outs))


def test_the_autograd_node_refuses_what_it_cannot_do():
    q, k, wq, wk, dq, dk = _inputs((5,), 4, 2, 64, torch.float32, seed=7)
    cos, sin = _tables(5, 64)
    wq.requires_grad_()
    (g,) = torch.autograd.grad(_call(q, k, wq, wk, cos, sin)[0].square().sum(), wq, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    with pytest.raises(RuntimeError, match="batched gradients"):
        torch.autograd.grad(_call(q, k, wq, wk, cos, sin)[0], wq, torch.ones(2, *q.shape, device="cuda"), is_grads_batched=True)
    y = _call(q, k, wq, wk, cos, sin)[0]
    q.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals():
    q, k, wq, wk, _, _ = _inputs((5,), 4, 2, 64, torch.float32)
    cos, sin = _tables(5, 64)
    pos = torch.zeros(5, dtype=torch.int64, device="cuda")
    for args, msg in (((q, k[:4], wq, wk, cos, sin), "expected q"), ((q, k[..., :32], wq, wk, cos, sin), "expected q"), ((q[0], k[0], wq, wk, cos, sin), "expected q"), ((q, k.half(), wq, wk, cos, sin), "share a dtype"),
                      ((q.double(), k.double(), wq, wk, cos, sin), "share a dtype"), ((q, k, wq.half(), wk, cos, sin), "weights must be"), ((q, k, wq, wk[:32], cos, sin), "weights must be"),
                      ((q, k, wq, wk, cos[:, :16], sin[:, :16]), "cos/sin"), ((q, k, wq, wk, cos[:4], sin[:4]), "cos/sin"), ((q, k, wq, wk, cos.double(), sin.double()), "cos/sin"), ((q, k, wq, wk, cos, sin[:4]), "cos/sin"),
                      ((q, k, wq, wk, cos, sin, pos[:4]), "one value for each token"), ((q, k, wq, wk, cos, sin, pos.float()), "int64 or int32"), ((q, k, wq, wk, cos.cpu(), sin), "same device"),
                      ((q, k, wq, wk, cos, sin, pos.cpu()), "same device|CUDA"), ((q, k, wq, wk, cos[:0], sin[:0], pos), "no rows"), ((q[..., :24], k[..., :24], wq[:24], wk[:24], cos[:, :12], sin[:, :12]), "multiple of 16")):
        with pytest.raises((RuntimeError, IndexError), match=msg):
            _call(*args)


def test_on_another_stream_and_captured_into_a_graph():
    from nanonemo_amd.kernels.hip import host

    print("\n[case] qk_norm on a side stream and in a graph", flush=True)
    q, k, wq, wk, dq, dk = _inputs((2000,), 12, 4, 64, torch.bfloat16, seed=8)
    cos, sin = _tables(100, 64)
    pos = torch.randint(0, 100, (2000,), device="cuda")

    def both():
        return *host().qk_norm_fwd(q, k, wq, wk, cos, sin, pos, EPS), *host().qk_norm_bwd(dq, dk, q, k, wq, wk, cos, sin, pos, EPS)

    ref = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = both()
    for i in range(4):
        for t in (q, k, dq, dk, wq, wk):
            t.copy_(torch.randn_like(t))
        pos.copy_(torch.randint(0, 100, pos.shape, device="cuda"))
        for t in outs:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, both())), i


def test_offsets_past_32_bits():
    print("\n[case] qk_norm of 2.9 million tokens", flush=True)
    T, H, KVH, D = 2_900_000, 12, 4, 64
    tail = _inputs((100,), H, KVH, D, torch.bfloat16, seed=9)
    wq, wk = tail[2:4]
    cos, sin = _tables(100, D)
    q, k, dq, dk = (torch.zeros(T, n, D, dtype=torch.bfloat16, device="cuda") for n in (H, KVH, H, KVH))
    assert (T - 100) * H * D > 2**31
    for t, x in zip((q, k, dq, dk), (tail[0], tail[1], tail[4], tail[5])):
        t[-100:] = x
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    pos[-100:] = torch.arange(100, device="cuda")
    outs = []
    for ins, p, g in (((q, k), pos, (dq, dk)), (tail[:2], pos[-100:], tail[4:])):
        leaves = [t.detach().requires_grad_() for t in (*ins, wq, wk)]
        y = _call(*leaves, cos, sin, p)
        outs.append([t.detach()[-100:] for t in y] + [t[-100:] if t.dim() > 1 else t for t in torch.autograd.grad(y, leaves, g)])
    for a, b in zip(outs[0][:4], outs[1][:4]):
        assert torch.equal(a, b)
    for a, b in zip(outs[0][4:], outs[1][4:]):  # zeros add nothing; the fp32 sums' order goes by the size: 400 or 1200 terms
        torch.testing.assert_close(a, b, rtol=0, atol=1200 * 2**-24 * 4 * b.abs().max().item())


def _layer(B, T, H, KVH, hd, lengths=None, **kw):
    """An attention layer with norms, whose weights are not ones, and what it is called with beside x."""
    from nanonemo_amd.kernels.hip.packed import Packing
    from tests.test_layers_gpu import _attention

    m, (cos, sin) = _attention(H, KVH, hd, T, rope_kernel="hip", qk_norm=True, **kw)
    g = torch.Generator(device="cuda").manual_seed(5)
    with torch.no_grad():
        for n in (m.q_norm, m.k_norm):
            n.weight.copy_(1 + 0.3 * torch.randn(hd, device="cuda", generator=g))
    if lengths is None:
        return m, (cos, sin)
    packing = Packing(lengths, H, KVH)
    return m, (cos[packing.positions], sin[packing.positions], packing)


def _layer64(x, cos, sin, H, KVH, eps, wq, wk, wv, wo, wqn, wkn):
    _, T, _ = x.shape
    c, s = cos[:T, None].double(), sin[:T, None].double()

    def rot(t, w):
        a, b = (w * t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps)).chunk(2, -1)
        return torch.cat((a * c - b * s, a * s + b * c), -1).transpose(1, 2)

    q, k, v = ((x @ w.t()).view(*x.shape[:2], h, -1) for w, h in ((wq, H), (wk, KVH), (wv, KVH)))
    q, k, v = rot(q, wqn), rot(k, wkn), v.transpose(1, 2)
    k, v = (t.repeat_interleave(H // KVH, 1) for t in (k, v))
    future = torch.ones(T, T, dtype=torch.bool, device=x.device).triu(1)
    p = ((q @ k.transpose(2, 3).contiguous()) / q.shape[-1] ** 0.5).masked_fill(future, -float("inf")).softmax(-1)
    return (p @ v).transpose(1, 2).reshape(*x.shape[:2], -1) @ wo.t()


def _parts(m):
    return m.wq.weight, m.wk.weight, m.wv.weight, m.wo.weight, m.q_norm.weight, m.k_norm.weight


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B, T, H, KVH, hd, lengths", [(2, 200, 12, 4, 64, None), (3, 65, 2, 2, 64, None), (1, 700, 8, 2, 32, None),
                                                       (1, 458, 12, 4, 64, [100, 1, 260, 0, 64, 33]), (1, 196, 4, 1, 32, [130, 1, 65])])
def test_attention_layer_with_norms_matches_float64(B, T, H, KVH, hd, lengths, dtype):
    from tests.test_layers_gpu import _modules_only, _rel

    print(f"\n[case] attention layer with norms B={B} T={T} H={H} KVH={KVH} hd={hd} {lengths} {dtype}", flush=True)
    m, more = _layer(B, T if lengths is None else max(lengths), H, KVH, hd, lengths)
    x = torch.randn(B, T, H * hd, device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(B, T, H * hd, device="cuda").to(dtype)

    def run(mod):
        with torch.autocast("cuda", dtype=dtype):
            y = mod(x, *more)
        return y, (y.detach(), *torch.autograd.grad(y, (x, *_parts(mod)), dy))

    y, got = run(m)
    node = y.grad_fn
    while "View" in node.name():
        node = node.next_functions[0][0]
    assert node.name() == "_AttentionLayerBackward"
    ref = run(_modules_only(m))[1]
    ins = [t.detach().double().requires_grad_() for t in (x, *_parts(m))]
    if lengths is None:
        y = _layer64(ins[0], *more, H, KVH, m.q_norm.eps, *ins[1:])
    else:
        i = lengths.index(max(lengths))
        c, s = (t.split(lengths)[i] for t in more[:2])
        y = torch.cat([_layer64(t, c, s, H, KVH, m.q_norm.eps, *ins[1:]) for t in ins[0].split(lengths, 1) if t.shape[1]], 1)
    exact = (y.detach(), *torch.autograd.grad(y, ins, dy.double()))
    # The 16-bit roundings on the longest path, each of u in the 2-norm, as the layer without norms has them (the norm rounds with
    # the rotation): weights, product, rotation of q and of k; P and O; the output weight, dO, dS, dq or dk, its rotation. And no
    # term may be worse than in the modules, which round more; but the 2-norm of n independent errors of equal size is itself only
    # within 1 / sqrt(2 n) of its mean (one standard deviation), the ratio of two within 1 / sqrt(n): four of those are allowed, 0.5
    # for the norms' 64 weights and 0.01 for the other tensors.
    u = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-11
    for name, a, b, e in zip(("y", "dx", "dwq", "dwk", "dwv", "dwo", "dq_norm", "dk_norm"), got, ref, exact):
        mine, theirs = _rel(a, e), _rel(b, e)
        print(f"  {name}: {mine:.2e}, modules {theirs:.2e}, bound {13**0.5 * u:.2e}", flush=True)
        assert mine <= 13**0.5 * u, name
        assert mine <= (1.1 + 4 * a.numel() ** -0.5) * theirs, name
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        assert torch.equal(m(x, *more), got[0])


@pytest.mark.parametrize("lengths", [None, [70, 30, 40]])
def test_attention_layer_with_norms_frozen_parts_and_repeated_backward(lengths):
    m, more = _layer(1, 140, 4, 2, 64, lengths)
    x = torch.randn(1, 140, 256, device="cuda", requires_grad=True)  # fp32 in, cast by the layer

    def loss():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return m(x, *more).float().square().sum()

    y = loss()
    y.backward(retain_graph=True)
    all_ = (x, *_parts(m))
    first = [t.grad.clone() for t in all_]
    y.backward()
    for a, t in zip(first, all_):
        assert torch.equal(a + a, t.grad)
    for i in range(len(all_)):  # each alone: the others' gradients are not formed
        for j, t in enumerate(all_):
            t.requires_grad_(i == j)
        (g,) = torch.autograd.grad(loss(), all_[i])
        assert torch.equal(g, first[i]), i


@pytest.mark.parametrize("lengths", [None, [20, 13]])
def test_attention_layer_with_norms_recorded_backward(lengths):
    from tests.test_layers_gpu import _modules_only

    m, more = _layer(1, 33, 4, 2, 32, lengths)
    x = torch.randn(1, 33, 128, device="cuda", requires_grad=True)
    out = []
    for mod in (m, _modules_only(m)):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = mod(x, *more)
        gs = torch.autograd.grad(y.float().sum(), (x, *_parts(mod)), create_graph=True)
        out.append([*(g.detach() for g in gs), *torch.autograd.grad(gs[4].square().sum(), x)])  # (through wo's gradient)
    for a, b in zip(*out):
        torch.testing.assert_close(a, b, rtol=5e-2, atol=5e-2 * b.abs().max().item())


def test_norms_with_hooks_are_called():
    """A hook on a head norm, another norm in its place, or its weight in another type, runs as a module."""
    from nanonemo_amd.model import RMSNorm

    m, more = _layer(1, 40, 4, 2, 64)
    x = torch.randn(1, 40, 256, device="cuda").bfloat16()

    def run():
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            return m(x, *more)

    plain, seen = run(), []
    h = m.k_norm.register_forward_hook(lambda _, ins, out: seen.append(out.shape))
    hooked = run()
    assert seen == [(1, 40, 2, 64)]
    h.remove()
    u = 2.0**-8  # one rounding more of q and of k: each of their scores' terms and its sum at random
    assert (hooked.float() - plain.float()).norm() <= 4 * u * plain.float().norm()
    assert torch.equal(run(), plain)

    class Half(RMSNorm):
        def forward(self, t):
            return 0 * super().forward(t)

    m.q_norm = Half(64, 1e-5).cuda()
    uniform = run()  # queries of zeros: the mean of the values so far
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        v = m.wv(x).view(1, 40, 2, 64).float()
        mean = (v.cumsum(1) / torch.arange(1, 41, device="cuda").view(1, 40, 1, 1)).repeat_interleave(2, 2).bfloat16()
        want = m.wo(mean.view(1, 40, 256)).float()
    assert (uniform.float() - want).norm() <= 3 * u * want.norm()


def test_attention_layer_with_norms_refuses_norms_of_other_sizes():
    from nanonemo_amd.kernels.hip import host

    m, (cos, sin) = _layer(1, 40, 4, 2, 64)
    x = torch.randn(40, 256, device="cuda").bfloat16()
    call = (x, cos, sin, 1, 40, 4, 2, m.wq.weight, m.wk.weight, m.wv.weight, m.wo.weight, False, None, None)
    good = m.q_norm.weight
    for bad in ((good[:32], good), (good, good.half()), (good.cpu(), good), (good, None)):
        with pytest.raises(RuntimeError):
            host().attention_layer_fwd(*call, *bad, 1e-5)
