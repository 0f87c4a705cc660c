"""GPU tests of the distillation kernels (kernels/hip/distill.py): a teacher's top logits, the loss and its gradient, and a
student's training step on them."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
INF, NAN = float("inf"), float("nan")

# The relative error of a row's fp32 sum of exponentials: an exponent's difference and product are rounded (2^-24 each, of at
# most about 20 for terms that count), exp2 is off by one step, and a thread adds at most some 50 terms before the join.
SUM = 1e-5


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- the top logits -----------------------------------------------------------------------------


def _logits(kind: str, rows: tuple, V: int, dtype, g) -> torch.Tensor:
    x = 2.5 * torch.randn(*rows, V, generator=g, device="cuda")
    if kind == "ties":
        x = x.round()
    elif kind == "constant":
        x = torch.full_like(x, 0.25)
    elif kind == "masked":  # all but a few at the type's lowest value or -inf, and rows with nothing else
        lowest = torch.finfo(dtype).min
        x = torch.where(torch.rand(x.shape, generator=g, device="cuda") < 0.02, x, torch.where(x > 0, lowest, -INF))
        x.view(-1, V)[0] = -INF
    elif kind == "zeros":
        x = torch.where(torch.rand(x.shape, generator=g, device="cuda") < 0.5, 0.0, -0.0)
    elif kind == "special":
        pick = torch.rand(x.shape, generator=g, device="cuda")
        x = torch.where(pick < 0.01, NAN, torch.where(pick < 0.02, INF, torch.where(pick < 0.03, -INF, x)))
        x.view(-1, V)[0, 0] = -NAN
    elif kind == "ascending":
        x = x.sort(-1).values
    elif kind == "spread":
        x = x * 40
    return x.to(dtype)


def _top64(x, k, tau):
    # (torch.sort has a NaN whose sign bit is set below everything; one sign for all of them)
    order = torch.sort(torch.where(x.isnan(), NAN, x.double() + 0.0), dim=-1, descending=True, stable=True)
    tail = order.values[..., k:] / tau
    rest = tail.logsumexp(-1) if tail.shape[-1] else torch.full(x.shape[:-1], -INF, dtype=torch.float64, device="cuda")
    return order.values[..., :k], order.indices[..., :k], rest


def _check_top(x, k, tau, what):
    from nanonemo_amd.kernels.hip.distill import top_logits

    v, i, r = top_logits(x, k, tau)
    rv, ri, rr = _top64(x, k, tau)
    assert v.dtype == x.dtype and i.dtype == torch.int64 and r.dtype == torch.float32, what
    assert torch.equal(i, ri), what
    assert torch.equal(v.double().nan_to_num(1e300), rv.nan_to_num(1e300)), what
    # (a type's lowest value over 0.7 lies outside fp32: -inf is its rounding)
    assert torch.equal(r.isnan(), rr.isnan()) and torch.equal(r.isinf(), rr.float().isinf()), what
    fine = rr.float().isfinite()
    assert ((r.double() - rr)[fine].abs() <= SUM + 2**-24 * rr[fine].abs()).all(), what


# Vocabularies around a group of 16 bytes and the kernels' row lengths (2048, 8192 and 65536 values), odd ones among them.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 64, 511, 1003, 2047, 2048, 2049, 8192, 8197, 32000, 50304, 60001, 65537, 131075])
def test_top_logits(V, dtype):
    for kind in ("normal", "ties", "ascending", "spread"):
        for k in sorted({1, min(2, V), min(7, V), min(64, V), min(200, V), min(512, V)}):
            print(f"\n[case] top logits V={V} k={k} {kind} {dtype}", flush=True)
            _check_top(_logits(kind, (3,), V, dtype, _gen(V + k)), k, 1.0 if k % 2 else 2.0, (kind, k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [5, 300, 700, 2500, 9000, 50304, 140001])
@pytest.mark.parametrize("kind", ["constant", "masked", "zeros", "special"])
def test_top_logits_of_equal_masked_and_special_values(kind, V, dtype):
    for k in sorted({1, min(4, V), min(33, V), min(300, V)}):
        print(f"\n[case] top logits V={V} k={k} {kind} {dtype}", flush=True)
        _check_top(_logits(kind, (4,), V, dtype, _gen(V + k)), k, 0.7, k)


def test_top_logits_where_the_rest_is_far_below():
    # The k-th value stands far above the others: their sum must not vanish.
    for V in (300, 50304):
        x = torch.randn(2, V, device="cuda")
        x[:, 5:9] += 400
        x[1, 9:] -= 1e4
        for k in (2, 4, 5):
            _check_top(x, k, 1.0, (V, k))


def test_top_logits_of_strided_rows_and_shapes():
    from nanonemo_amd.kernels.hip.distill import top_logits

    x = torch.randn(3, 6, 1003, device="cuda").bfloat16()
    for t in (x, x[:, :-1], x[:, 1:], x[::2], x.transpose(0, 1), x[..., 1:], x[..., ::2], x[0, 0], x[:0], x[1:2, 2:3], x[:, :1].expand(3, 4, 1003), x.view(3, 2, 3, 1003)[:, :, 1:],
              x[:, ::2], x.view(3, 2, 3, 1003).transpose(0, 2)):
        got, ref = top_logits(t, 9, 2.0), _top64(t, 9, 2.0)
        assert got[0].shape == ref[0].shape and torch.equal(got[1], ref[1]) and torch.equal(got[0].double(), ref[0])
        assert ((got[2].double() - ref[2]).abs() <= SUM + 2**-24 * ref[2].abs()).all()


# ---- the loss -----------------------------------------------------------------------------------


def _reference(z, v, idx, rest, y, tau, w, grad=1.0):
    """(loss, gradient, how far the loss and the gradient may be off) in fp64, rows flattened."""
    V = z.shape[-1]
    half, tiny = torch.finfo(z.dtype).eps / 2, torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps + 1e-37
    x = z.detach().double().reshape(-1, V).requires_grad_()
    idx = idx.reshape(len(x), -1)
    keep = torch.ones(len(x), dtype=torch.bool, device="cuda") if y is None else y.reshape(-1) != -100
    t = v.double().reshape(len(x), -1) / tau
    logq = torch.log_softmax(x / tau, -1)
    on = logq.gather(-1, idx)
    others = torch.ones_like(logq, dtype=torch.bool).scatter_(-1, idx, False)
    q_rest = (logq.exp() * others).sum(-1, keepdim=True).detach()
    p_rest = torch.zeros_like(q_rest)
    if rest is not None:
        t = torch.cat((t, rest.double().reshape(-1, 1)), -1)
        on = torch.cat((on, logq.masked_fill(~others, -INF).logsumexp(-1, keepdim=True)), -1)
    p = torch.softmax(t, -1)
    if rest is not None:
        p_rest = p[:, -1:]
    hard = y is not None and w < 1
    row = w * tau**2 * torch.where(p > 0, p * (torch.log_softmax(t, -1) - on), 0.0).sum(-1) if w else torch.zeros(len(x), dtype=torch.float64, device="cuda")
    if hard:
        s = torch.log_softmax(x, -1)
        row = row - (1 - w) * s.gather(-1, y.reshape(-1, 1).clamp_min(0)).squeeze(-1)
    n = keep.sum()
    loss = torch.where(keep, row, 0.0).sum() / n
    (d,) = torch.autograd.grad(loss, x, torch.tensor(grad, device="cuda").double())  # (as the kernel is given it)
    # an error of the row's sum reaches KL times q_rest - p_rest, and the cross entropy at most once
    off = w * tau**2 * (q_rest - p_rest).abs().squeeze(-1) + (1 - w if hard else 0.0)
    loss_off = SUM * (off * keep).sum() / n + 2**-23 * loss.detach().abs() + 1e-12
    q = logq.detach().exp()
    # (q p_rest / q_rest as a share of the rest: q and q_rest may both vanish, even in fp64)
    share = torch.where(others & (p_rest > 0), p_rest * torch.softmax(logq.detach().masked_fill(~others, -INF), -1), 0.0).nan_to_num(0.0)
    size = w * tau * (q + share) + ((1 - w) * s.detach().exp() if hard else 0.0)
    slack = SUM * size * (keep / n * abs(grad)).unsqueeze(-1)
    return loss.detach(), d.view(z.shape), loss_off, (half * (d.abs() + slack) + slack + tiny).view(z.shape)


def _check_loss(z, v, idx, rest, y, tau, w, what, grad=1.0):
    from nanonemo_amd.kernels.hip.distill import distill_loss

    z = z.detach().requires_grad_()
    loss = distill_loss(z, v, idx, rest, y, tau, w)
    (d,) = torch.autograd.grad(loss, z, torch.tensor(grad, device="cuda"))
    rl, rd, loss_off, off = _reference(z, v, idx, rest, y, tau, w, grad)
    assert loss.dtype == torch.float32 and loss.shape == () and d.dtype == z.dtype and d.shape == z.shape, what
    assert abs(loss.item() - rl.item()) <= loss_off.item(), what
    worst = ((d.double() - rd).abs() / off).max().item()
    assert worst <= 1.0, what


def _case(rows, V, k, dtype, tau, g, near=1.0):
    z = 2 * torch.randn(*rows, V, generator=g, device="cuda")
    t = z + near * torch.randn(*rows, V, generator=g, device="cuda")
    v, idx = t.topk(k, dim=-1)
    rest = (t / tau).scatter(-1, idx, -INF).logsumexp(-1)
    y = torch.randint(0, V, rows, generator=g, device="cuda")
    y = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.4, idx[..., 0], y)
    return z.to(dtype), v.to(dtype), idx, rest, y


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, V, k", [((1,), 1, 1), ((2,), 2, 1), ((3,), 7, 7), ((2, 3), 9, 4), ((5,), 64, 8), ((1, 37), 1003, 7), ((3, 4), 2048, 64), ((7,), 2049, 65), ((2, 2), 8197, 512), ((9,), 50304, 64),
                                        ((2,), 131075, 100), ((1,), 393216, 300)])
def test_distill_loss_and_gradient_match_float64(rows, V, k, dtype):
    g = _gen(V + k)
    for tau in (1.0, 2.0, 0.7):
        z, v, idx, rest, y = _case(rows, V, k, dtype, tau, g)
        if y.numel() > 2:
            y.view(-1)[1] = -100
        if k == V:
            rest = None  # there is no rest
        for r, t, w in ((None, None, 1.0), (rest, None, 1.0), (None, y, 0.5), (rest, y, 0.5), (rest, y, 1.0), (rest, y, 0.0), (None, y, 0.9)):
            print(f"\n[case] distill rows={rows} V={V} k={k} {dtype} tau={tau} rest={r is not None} targets={t is not None} weight={w}", flush=True)
            _check_loss(z, v, idx, r, t, tau, w, (tau, r is not None, t is not None, w), 0.6)


@pytest.mark.parametrize("tau", [1.0, 4.0])
@pytest.mark.parametrize("near", [0.3, 0.01, 0.001])
def test_a_student_near_its_teacher(near, tau):
    # The loss is then far below the logits' logsumexp (down to 1e-7): the bound of _reference shrinks with it.
    z, v, idx, rest, y = _case((4, 8), 5000, 20, torch.float32, tau, _gen(3), near)
    _check_loss(z, v, idx, rest, None, tau, 1.0, near)
    _check_loss(z, v, idx, rest, y, tau, 0.5, near)


def test_teacher_types_orders_and_scales():
    g = _gen(5)
    z, v, idx, rest, y = _case((2, 9), 3001, 40, torch.bfloat16, 2.0, g)
    order = torch.rand(idx.shape, generator=g, device="cuda").argsort(-1)  # any order of the k
    for dt in DTYPES:
        _check_loss(z, v.to(dt).gather(-1, order), idx.gather(-1, order), rest, y, 2.0, 0.5, dt)
    _check_loss(z, v - 1000.0, idx, rest - 500.0, y, 2.0, 0.5, "a teacher's shift")  # (values in bf16 keep their differences to 4)
    _check_loss((z.float() + 3000).half().float(), v, idx, rest, y, 2.0, 0.5, "a student's shift")
    vm = v.clone()
    vm[..., 30:] = -INF  # a teacher that gives fewer than k
    _check_loss(z, vm, idx, rest, y, 2.0, 0.5, "fewer")
    _check_loss(z, v, idx, torch.full_like(rest, -INF), y, 2.0, 0.5, "nothing in the rest")


@pytest.mark.parametrize("V", [300, 5000])
def test_a_student_whose_top_set_stands_far_above_or_below_the_rest(V):
    # 300 above: the rest's probabilities vanish in fp32 beside the top set's, its shares of the rest's gradient do not. 300
    # below (and 900, past the exponents that fp32 sums reach): the top set's vanish.
    g = _gen(13)
    z, v, idx, rest, y = _case((6,), V, 9, torch.float32, 1.0, g)
    for up in (300.0, -300.0, 900.0, -900.0):
        x = z.scatter_add(-1, idx, torch.full_like(v, up))
        y[0] = next(j for j in range(V) if j not in idx[0].tolist())
        for r, t, w in ((rest, None, 1.0), (rest, y, 0.5), (None, y, 0.5)):
            _check_loss(x, v, idx, r, t, 1.0, w, (up, r is not None, w))
    # a masked vocabulary: all but the top set at the type's lowest value, or gone
    low = torch.full_like(z, torch.finfo(z.dtype).min / 4).scatter(-1, idx, z.gather(-1, idx))
    _check_loss(low, v, idx, None, None, 1.0, 1.0, "lowest")
    _check_loss(low.masked_fill(low < -1e30, -INF), v, idx, None, None, 1.0, 1.0, "gone")
    _check_loss(low, v, idx, torch.full_like(rest, -INF), None, 1.0, 1.0, "lowest, nothing in the rest")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [300, 5000])
def test_a_masked_vocabulary_at_any_level(V, dtype):
    # All but the top set at -inf, and what is left far below (or above) 0: the gradient of the rest is 0, not 0 times e^100.
    z, v, idx, rest, y = _case((6,), V, 9, torch.float32, 0.5, _gen(29))
    y = idx[..., 3].clone()
    other = next(j for j in range(V) if not (idx == j).any())
    for level in (-300.0, 300.0):
        gone = torch.full_like(z, -INF).scatter(-1, idx, z.gather(-1, idx) + level).to(dtype)
        for tau in (0.5, 1.0, 2.0):
            for t, w in ((None, 1.0), (y, 0.5), (y, 0.0)):
                print(f"\n[case] masked V={V} {dtype} level={level} tau={tau} weight={w}", flush=True)
                _check_loss(gone, v, idx, None, t, tau, w, ("gone", level, tau, w))
        # the target as the only one of the rest, near the top set or far below it
        for below in (2.0, 150.0):
            alone = gone.clone()
            alone[..., other] = level - below
            for r in (None, rest):
                print(f"\n[case] masked but the target V={V} {dtype} level={level} below={below} rest={r is not None}", flush=True)
                _check_loss(alone, v, idx, r, torch.full_like(y, other), 0.5, 0.5, ("alone", level, below, r is not None))


def test_strided_logits_and_teachers():
    g = _gen(6)
    z, v, idx, rest, y = _case((3, 6), 1003, 9, torch.bfloat16, 2.0, g)
    wide = torch.randn(3, 7, 1003, device="cuda").bfloat16()
    wide[:, :-1] = z
    _check_loss(wide[:, :-1], v, idx, rest, y, 2.0, 0.5, "a view")
    _check_loss(wide[:, :-1], v.transpose(-1, -2).contiguous().transpose(-1, -2), idx.transpose(0, 1).contiguous().transpose(0, 1), torch.stack((rest, rest), -1)[..., 0],
                torch.stack((y, y), -1)[..., 1], 2.0, 0.5, "strided teachers")
    _check_loss(z[..., ::2], v, idx // 2, rest, y // 2, 2.0, 1.0, "strided values") if not _twice(idx // 2) else None
    _check_loss(z[0, 0], v[0, 0], idx[0, 0], rest[0, 0], y[0, 0], 2.0, 0.5, "one row")
    _check_loss(z[:, :1].expand(3, 6, 1003), v, idx, rest, y, 2.0, 0.5, "expanded")


def _twice(idx):
    s = idx.sort(-1).values
    return bool((s[..., 1:] == s[..., :-1]).any())


@pytest.mark.parametrize("V", [50, 3000])
def test_an_index_that_is_there_twice_adds_up(V):
    # As a sum over entries has it: the reference gathers and scatters entry by entry.
    g = _gen(7)
    z, v, idx, rest, y = _case((6,), V, 12, torch.float32, 2.0, g)
    idx[:, 5] = idx[:, 2]
    idx[1:, 11] = idx[1:, 2]
    idx[2, :] = idx[2, 0]
    y[3], y[4] = idx[3, 2], idx[4, 7]
    for r, t, w in ((None, None, 1.0), (rest, None, 1.0), (rest, y, 0.5)):
        _check_loss(z, v, idx, r, t, 2.0, w, w)


def test_rows_that_do_not_count_and_values_out_of_range():
    from nanonemo_amd.kernels.hip.distill import distill_loss

    g = _gen(8)
    for V in (300, 3000):
        z, v, idx, rest, y = _case((4, 5), V, 6, torch.float32, 1.0, g)
        y[1] = -100
        zp, vp, ip, rp = z.clone(), v.clone(), idx.clone(), rest.clone()
        zp[1], vp[1], ip[1], rp[1] = NAN, INF, -7, NAN  # what a padded row holds does not matter
        for w in (1.0, 0.5):
            a, b = (t.requires_grad_() for t in (z.clone(), zp))
            la, lb = distill_loss(a, v, idx, rest, y, 1.0, w), distill_loss(b, vp, ip, rp, y, 1.0, w)
            (da,), (db,) = torch.autograd.grad(la, a), torch.autograd.grad(lb, b)
            assert torch.equal(la, lb) and torch.equal(da, db) and (db[1] == 0).all()
            for bad_i, bad_y in ((-1, None), (V, None), (1 << 40, None), (None, V), (None, -1)):
                i, t = idx.clone(), y.clone()
                if bad_i is not None:
                    i[2, 3, 4] = bad_i
                else:
                    t[2, 3] = bad_y
                x = z.clone().requires_grad_()
                loss = distill_loss(x, v, i, rest, t, 1.0, w)
                (d,) = torch.autograd.grad(loss, x)
                assert loss.isnan() and d[2, 3].isnan().all()
                d[2, 3] = 0
                assert d.isfinite().all()
        x = z.clone().requires_grad_()
        loss = distill_loss(x, v, idx, rest, torch.full_like(y, -100), 1.0, 0.5)
        assert loss.isnan() and (torch.autograd.grad(loss, x)[0] == 0).all()  # no row counts
    assert distill_loss(z[:0], v[:0], idx[:0], rest[:0], y[:0]).isnan()


def test_special_logits_show():
    from nanonemo_amd.kernels.hip.distill import distill_loss

    z, v, idx, rest, y = _case((4,), 500, 6, torch.float32, 1.0, _gen(9))
    other = next(j for j in range(500) if j not in idx[1].tolist() and j != y[1])
    for value in (NAN, INF, -INF):
        for at in (other, int(idx[1, 2]), int(y[1])):
            x = z.clone()
            x[1, at] = value
            x.requires_grad_()
            loss = distill_loss(x, v, idx, rest, y, 1.0, 0.5)
            (d,) = torch.autograd.grad(loss, x)
            if value == -INF and at == other:  # masked: no probability, no gradient
                rl, rd, loss_off, off = _reference(x, v, idx, rest, y, 1.0, 0.5)
                assert (loss.double() - rl).abs() <= loss_off and ((d.double() - rd).abs() <= off).all() and d[1, at] == 0
            elif value == -INF:
                assert loss == INF and d.isfinite().all()
            else:
                assert loss.isnan() and d[1].isnan().all()
            assert d[[0, 2, 3]].isfinite().all()


def test_rows_beyond_32_bit_offsets():
    from nanonemo_amd.kernels.hip.distill import distill_loss, top_logits

    print("\n[case] distill beyond 2^31 logits", flush=True)
    R, V = 43000, 50304
    z = torch.randn(R, V, device="cuda", dtype=torch.bfloat16)
    v, idx, rest = top_logits(z, 5, 2.0)
    rv, ri, rr = _top64(z[-2:], 5, 2.0)
    assert torch.equal(idx[-2:], ri) and torch.equal(v[-2:].double(), rv)
    y = torch.full((R,), -100, device="cuda")
    y[-2:], y[:2] = 7, 9
    z.requires_grad_()
    (d,) = torch.autograd.grad(distill_loss(z, v, idx, rest, y, 2.0, 0.5), z)
    part = torch.cat((z[:2], z[-2:])).detach().requires_grad_()
    at = torch.tensor([0, 1, R - 2, R - 1], device="cuda")
    (ref,) = torch.autograd.grad(distill_loss(part, v[at], idx[at], rest[at], y[at], 2.0, 0.5), part)
    assert torch.equal(d[at], ref) and not d[2:-2].any()


def test_op_and_eager_path_give_the_same_bits_and_the_ops_pass_opcheck():
    from nanonemo_amd.kernels.hip.distill import distill_loss, top_logits

    z, v, idx, rest, y = _case((2, 5), 700, 6, torch.float32, 2.0, _gen(10))
    z.requires_grad_()
    loss, op = distill_loss(z, v, idx, rest, y, 2.0, 0.5), torch.ops.nanonemo.distill_loss(z, v, idx, rest, y, 2.0, 0.5)[0]
    assert 'DistillNode' in loss.grad_fn.name() and torch.equal(loss, op)
    (d,) = torch.autograd.grad(loss, z, retain_graph=True)
    assert torch.equal(d, torch.autograd.grad(loss, z)[0]) and torch.equal(d, torch.autograd.grad(op, z)[0])
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(torch.ops.nanonemo.top_logits, (z.detach(), 4, 2.0))
    torch.library.opcheck(torch.ops.nanonemo.distill_loss, (z.detach(), v, idx, rest, y, 2.0, 0.5), test_utils=tests)
    with torch.no_grad():
        assert torch.equal(distill_loss(z, v, idx, rest, y, 2.0, 0.5), loss)
    f = torch.compile(lambda a: distill_loss(a * 1.0, *top_logits(a.flip(0), 6, 2.0), y, 2.0, 0.5), fullgraph=True, backend="aot_eager")
    eager = distill_loss(z * 1.0, *top_logits(z.flip(0), 6, 2.0), y, 2.0, 0.5)
    got = f(z)
    assert torch.equal(got, eager) and torch.equal(torch.autograd.grad(got, z)[0], torch.autograd.grad(eager, z)[0])


def test_the_autograd_node_refuses_what_it_cannot_do():
    from nanonemo_amd.kernels.hip.distill import distill_loss

    z, v, idx, rest, y = _case((4,), 60, 5, torch.float32, 1.0, _gen(14))
    z.requires_grad_()
    (g,) = torch.autograd.grad(distill_loss(z, v, idx), z, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    with pytest.raises(RuntimeError, match="batched gradients"):
        torch.autograd.grad(distill_loss(z, v, idx), z, torch.ones(2, device="cuda"), is_grads_batched=True)
    loss = distill_loss(z, v, idx)
    with torch.no_grad():
        z.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    loss = distill_loss(z, v, idx, rest, y, 1.0, 0.5)
    a, b = (torch.autograd.grad(loss * 2, z, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(a, b)
    assert torch.autograd.grad(distill_loss(z * 1.0, v, idx, rest, y, 1.0, 0.5) * 2, z)[0].equal(a)


def test_gradient_matches_differences():
    from nanonemo_amd.kernels.hip.distill import distill_loss

    # Central differences in the kernels' own loss: h = 2^-5 leaves a truncation of h^2/6 of the third derivative (at most
    # tau^2 / tau^3 + 1 of a row's share) and the loss's rounding over 2h.
    z, v, idx, rest, y = _case((3,), 40, 5, torch.float32, 2.0, _gen(11))
    z.requires_grad_()
    loss = distill_loss(z, v, idx, rest, y, 2.0, 0.5)
    (d,) = torch.autograd.grad(loss, z)
    h = 2.0**-5
    for j in [int(idx[0, 0]), int(y[0]), 0, 1, 2, 39]:
        e = torch.zeros_like(z)
        e[0, j] = h
        with torch.no_grad():
            num = (distill_loss(z + e, v, idx, rest, y, 2.0, 0.5) - distill_loss(z - e, v, idx, rest, y, 2.0, 0.5)) / (2 * h)
        assert abs(num - d[0, j]) <= h * h / 6 * 1.5 / 3 + 4 * 2**-24 * loss.item() / (2 * h) + 2 * SUM


def test_on_another_stream_and_captured_into_a_graph():
    from nanonemo_amd.kernels.hip import host
    from nanonemo_amd.kernels.hip.distill import distill_loss, top_logits

    print("\n[case] distill on a side stream and in a graph", flush=True)
    z = torch.randn(16, 5000, device="cuda").bfloat16()
    t = torch.randn(16, 5000, device="cuda").bfloat16()
    y = torch.randint(0, 5000, (16,), device="cuda")
    one = torch.ones((), device="cuda")

    def chain():
        v, idx, rest = top_logits(t, 20, 2.0)
        loss, stats = host().distill_fwd(z, v, idx, rest, y, 2.0, 0.5)
        return v, idx, rest, loss, host().distill_bwd(one, z, v, idx, y, stats, 2.0, 0.5)

    ref = chain()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    assert torch.equal(distill_loss(z, ref[0], ref[1], ref[2], y, 2.0, 0.5), ref[3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for i in range(4):
        z.copy_(torch.randn_like(z)), t.copy_(torch.randn_like(t)), y.random_(0, 5000)
        for o in got:
            o.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, chain())), i


SMALL = dict(n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, d_ff=512, vocab_size=512, max_seq_len=128, attn_backend="math_fp32")
HIP = dict(attn_kernel="hip_bthd", rope_kernel="hip", norm_kernel="hip", emb_kernel="hip")


def test_the_students_step_matches_the_plain_models():
    # Teacher, student, loss and gradients on this build's kernels against the same models on PyTorch's operations: the
    # teacher's logits are computed in bf16 either way, so both students are given the kernels' teacher.
    from nanonemo_amd.model import ModelConfig, NanoNemo
    from nanonemo_amd.train import make_optimizer, teacher_batches, train_step

    torch.manual_seed(1)
    teacher = NanoNemo(ModelConfig(**{**SMALL, "n_layers": 3}, **HIP)).cuda()
    for p in teacher.parameters():  # logits that differ
        p.data.mul_(2.0)
    idx = torch.randint(0, 512, (2, 128), device="cuda")
    y = idx.roll(-1, 1)
    y[:, 100:] = -100
    (batch,) = teacher_batches(teacher, [(idx, y)], 16, temperature=2.0, weight=0.5)
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        full = teacher(idx)[0]
    rv, ri, rr = _top64(full, 16, 2.0)
    assert torch.equal(batch[2].indices, ri) and torch.equal(batch[2].values.double(), rv) and ((batch[2].rest - rr).abs() <= SUM + 2**-24 * rr.abs()).all()
    out, models = [], []
    for kernels in ({}, HIP):
        torch.manual_seed(0)
        m = NanoNemo(ModelConfig(**SMALL, **kernels)).cuda()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            logits, loss = m(*batch)
        assert logits.shape == (2, 128, 512) and not batch[2].values.requires_grad
        loss.backward()
        out.append((loss.detach(), {n: p.grad for n, p in m.named_parameters()}))
        models.append(m)
    torch.testing.assert_close(out[1][0], out[0][0], rtol=5e-3, atol=5e-3)  # as the model's tests have it for bf16
    for n, r in out[0][1].items():
        torch.testing.assert_close(out[1][1][n], r, rtol=5e-2, atol=5e-2 * r.abs().max().item(), msg=n)
    m = models[1]
    before = m.tok_emb.weight.detach().clone()
    m.zero_grad()
    loss, norm = train_step(m, make_optimizer(m), [batch])
    assert loss.isfinite() and norm.isfinite() and not torch.equal(before, m.tok_emb.weight)


def test_a_compiled_student_matches_the_eager_one():
    from nanonemo_amd.model import ModelConfig, NanoNemo

    torch.manual_seed(2)
    m = NanoNemo(ModelConfig(**SMALL, **HIP)).cuda()
    idx = torch.randint(0, 512, (2, 128), device="cuda")
    y = idx.roll(-1, 1)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        teacher = m.teach(idx, 8, 2.0, 0.5)
    out = []
    for f in (m, torch.compile(m, fullgraph=True, backend="aot_eager")):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            _, loss = f(idx, y, teacher)
        out.append((loss.detach(), torch.autograd.grad(loss, tuple(m.parameters()))))
    # (eagerly the fused layers keep fp32 weight gradients, compiled the modules round them: the model tests' bounds for bf16)
    torch.testing.assert_close(out[1][0], out[0][0], rtol=5e-3, atol=5e-3)
    for a, b in zip(out[1][1], out[0][1]):
        torch.testing.assert_close(a, b, rtol=5e-2, atol=5e-2 * b.abs().max().item())


def test_refusals():
    from nanonemo_amd.kernels.hip.distill import distill_loss, top_logits

    z, v, idx, rest, y = _case((3,), 50, 4, torch.float32, 1.0, _gen(12))
    for call, error, msg in (
        (lambda: top_logits(z, 0), ValueError, "k must be"), (lambda: top_logits(z, 51), ValueError, "k must be"), (lambda: top_logits(torch.zeros(2, 600, device="cuda"), 513), ValueError, "k must be"),
        (lambda: top_logits(z, 4, 0.0), ValueError, "temperature"), (lambda: top_logits(z, 4, NAN), ValueError, "temperature"), (lambda: top_logits(z.double(), 4), RuntimeError, "float32 tensor"),
        (lambda: top_logits(torch.zeros(1, 393217, device="cuda"), 4), RuntimeError, "invalid sizes"),
        (lambda: distill_loss(z, v, idx, rest, y, 1.0, 1.5), ValueError, "weight"), (lambda: distill_loss(z, v, idx, rest, None, 1.0, 0.5), ValueError, "needs targets"),
        (lambda: distill_loss(z, v.requires_grad_(), idx), ValueError, "no gradient"), (lambda: distill_loss(z, v.detach()[:2], idx), RuntimeError, "logits' rows"),
        (lambda: distill_loss(z, v.detach(), idx.int()), RuntimeError, "int64"), (lambda: distill_loss(z, v.detach(), idx, rest.double()), RuntimeError, "rest must be"),
        (lambda: distill_loss(z, v.detach(), idx, rest[:2]), RuntimeError, "rest must be"), (lambda: distill_loss(z, v.detach(), idx, rest, y.int()), RuntimeError, "targets must be"),
        (lambda: distill_loss(z, v.detach(), idx, rest.cpu()), RuntimeError, "same device|CUDA"), (lambda: distill_loss(z.cpu(), v.detach(), idx), RuntimeError, "CUDA"),
    ):
        with pytest.raises(error, match=msg):
            call()


# ---- the whole range of temperatures ------------------------------------------------------------


def _check_loss_at(z, v, idx, rest, y, tau, w, what):
    """_check_loss with the rounding of fp64 added, which tau^2 makes count: the logsumexps, of terms up to `most` in size, are
    sums of k values and of at most 256 + 16 partial ones, on either side."""
    from nanonemo_amd.kernels.hip.distill import distill_loss

    z = z.detach().requires_grad_()
    loss = distill_loss(z, v, idx, rest, y, tau, w)
    (d,) = torch.autograd.grad(loss, z)
    rl, rd, loss_off, off = _reference(z, v, idx, rest, y, tau, w)
    most = 13 + max(t.abs().max().item() for t in (z.detach().double() / tau, v.double() / tau))
    loss_off = loss_off + w * tau**2 * 2 * (v.shape[-1] + 272) * 2.0**-53 * most
    assert abs(loss.item() - rl.item()) <= loss_off.item(), what
    assert d.isfinite().all(), what
    worst = ((d.double() - rd).abs() / off).max().item()
    assert worst <= 1.0, (what, worst)


@pytest.mark.parametrize("tau", [1e-4, 0.01, 0.05, 2.0, 3.0, 4.0, 8.0, 9.0, 10.0, 20.0, 100.0, 1e4])
@pytest.mark.parametrize("rows, V, k, dtype", [((1,), 512, 9, torch.float32), ((300,), 1003, 7, torch.float32), ((1,), 50304, 64, torch.float32), ((260,), 50304, 64, torch.bfloat16),
                                               ((2,), 393216, 100, torch.float32)])
def test_distill_loss_over_the_range_of_temperatures(rows, V, k, dtype, tau):
    # The logsumexp of z / tau times tau lies up to tau ln V above the logits, their softmax at temperature 1 does not.
    z, v, idx, rest, y = _case(rows, V, k, dtype, tau, _gen(V + k))
    if y.numel() > 2:
        y.view(-1)[1] = -100
    for r, t, w in ((rest, y, 0.5), (rest, y, 0.0), (None, y, 0.9), (rest, None, 1.0), (None, None, 1.0)):
        print(f"\n[case] distill rows={rows} V={V} k={k} {dtype} tau={tau} rest={r is not None} targets={t is not None} weight={w}", flush=True)
        _check_loss_at(z, v, idx, r, t, tau, w, (r is not None, t is not None, w))


@pytest.mark.parametrize("tau", [2.0, 4.0, 20.0])
def test_the_cross_entropys_gradient_of_logits_far_below(tau):
    # Probabilities down to 1e-30, of the cross entropy alone.
    z, v, idx, _, y = _case((5,), 3001, 9, torch.float32, tau, _gen(31))
    z[:, 100:200] -= 60.0
    _check_loss_at(z, v, idx, None, y, tau, 0.0, tau)


@pytest.mark.parametrize("tau", [1e-4, 0.01, 8.0, 100.0, 1e4])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [64, 1003, 5000, 50304, 140001])
def test_top_logits_over_the_range_of_temperatures(V, dtype, tau):
    print(f"\n[case] top logits V={V} {dtype} tau={tau}", flush=True)
    for k in (1, 33):
        _check_top(_logits("normal", (3,), V, dtype, _gen(V + k)), k, tau, k)


@pytest.mark.parametrize("V", [300, 5000])
def test_a_masked_top_set_at_any_level(V):
    # The top set at -inf, the others far below (or above) 0. A teacher with mass in the top set makes the loss infinite, one
    # with all its mass in the rest does not.
    z, v, idx, rest, y = _case((6,), V, 9, torch.float32, 1.0, _gen(37))
    y = torch.full_like(y, next(j for j in range(V) if not (idx == j).any()))
    for level in (-3000.0, -800.0, -300.0, 300.0):
        gone = (z + level).scatter(-1, idx, -INF)
        for tau in (0.5, 1.0, 2.0, 3.0):
            for values, r, t, w in ((v, rest, None, 1.0), (v, None, y, 0.5), (torch.full_like(v, -INF), rest, None, 1.0), (torch.full_like(v, -INF), rest, y, 0.5), (v, None, y, 0.0)):
                what = (level, tau, bool(values[0, 0] == -INF), r is not None, w)
                print(f"\n[case] masked top set V={V} {what}", flush=True)
                from nanonemo_amd.kernels.hip.distill import distill_loss

                x = gone.clone().requires_grad_()
                loss = distill_loss(x, values, idx, r, t, tau, w)
                (d,) = torch.autograd.grad(loss, x)
                rl, rd, loss_off, off = _reference(x, values, idx, r, t, tau, w)
                assert rl.isfinite() == bool(w == 0 or values[0, 0] == -INF), what
                assert loss.item() == rl.item() or abs(loss.item() - rl.item()) <= loss_off.item(), what
                assert ((d.double() - rd).abs() <= off).all(), what


@pytest.mark.parametrize("V", [131072, 393216])
def test_a_rest_of_one_logit_and_very_many_below_fp32s_exponents(V):
    # e^-66.5 and some hundred thousand times e^-88, which fp32's normal numbers do not reach: 4e-5 to 2e-4 of the rest.
    z = torch.full((2, V), -88.0, device="cuda")
    z[:, 5:13] = torch.linspace(0.0, 1.0, 8, device="cuda")
    z[:, 77] = -66.5
    _check_top(z, 8, 1.0, V)
    _check_top(4 * z, 8, 4.0, V)
    idx = torch.arange(5, 13, device="cuda").expand(2, 8).contiguous()
    v, y = z.gather(-1, idx), torch.full((2,), 5, device="cuda")
    for tau in (1.0, 2.0, 4.0, 3.0):
        for t, w in ((None, 1.0), (y, 0.5)):
            print(f"\n[case] a rest of one logit V={V} tau={tau} weight={w}", flush=True)
            _check_loss(tau * z, tau * v, idx, torch.ones(2, device="cuda"), t, tau, w, (tau, w))


@pytest.mark.parametrize("V", [300, 5000])
@pytest.mark.parametrize("tau", [1.0, 2.0, 5.0])
def test_a_teachers_rest_where_the_student_has_none(V, tau):
    # Infinite divergence; the gradient is that of the top set's terms, and 0 where nothing is left.
    from nanonemo_amd.kernels.hip.distill import distill_loss

    z, v, idx, rest, y = _case((6,), V, 9, torch.float32, tau, _gen(41))
    x = torch.full_like(z, -INF).scatter(-1, idx, z.gather(-1, idx))
    p = torch.softmax(torch.cat((v.double() / tau, rest.double().unsqueeze(-1)), -1), -1)[:, :-1]
    on = x.double().gather(-1, idx)
    for t, w in ((None, 1.0), (idx[:, 3].clone(), 0.5)):
        x = x.detach().requires_grad_()
        loss = distill_loss(x, v, idx, rest, t, tau, w)
        (d,) = torch.autograd.grad(loss, x)
        ref = w * tau * (torch.softmax(on / tau, -1) - p)
        if t is not None:
            ref = ref + (1 - w) * (torch.softmax(on, -1) - (idx == t.unsqueeze(-1)).double())
        assert loss == INF and (d.scatter(-1, idx, 0.0) == 0).all()
        # (fp64 throughout, rounded once)
        assert ((d.gather(-1, idx).double() - ref / 6).abs() <= 2**-24 * (ref / 6).abs() + 1e-14).all()


def test_a_model_with_kernels_distils_what_they_do_not_take():
    # k above 512, a vocabulary above 393216, a teacher in fp64: the PyTorch form, as a model without kernels has it.
    from nanonemo_amd.model import ModelConfig, NanoNemo

    for vocab, k, dtype in ((700, 600, None), (393300, 5, None), (512, 7, torch.float64)):
        print(f"\n[case] model vocab={vocab} k={k} values {dtype}", flush=True)
        out = []
        for kernels in ({}, dict(norm_kernel="hip")):
            torch.manual_seed(3)
            m = NanoNemo(ModelConfig(**{**SMALL, "n_layers": 1, "d_model": 64, "d_ff": 64, "n_heads": 2, "n_kv_heads": 1, "vocab_size": vocab}, **kernels)).cuda()
            idx = torch.randint(0, vocab, (1, 16), generator=torch.Generator().manual_seed(1)).cuda()
            t = m.teach(idx, k, 2.0, 0.5)
            if dtype is not None:
                t = t._replace(values=t.values.to(dtype), rest=t.rest.to(dtype))
            _, loss = m(idx, idx.roll(-1, 1), t)
            out.append((t, loss, torch.autograd.grad(loss, m.tok_emb.weight)[0]))
        assert out[1][0].values.shape == (1, 16, k)
        for a, b in ((out[1][0].values, out[0][0].values), (out[1][0].rest, out[0][0].rest), (out[1][1], out[0][1]), (out[1][2], out[0][2])):
            torch.testing.assert_close(a, b, rtol=1e-3, atol=1e-5)  # (the norms alone differ, by fp32 roundings)
    with pytest.raises(ValueError, match="k must be"):
        m.teach(idx, 0)
    with pytest.raises(ValueError, match="temperature"):
        m.teach(idx, 4, -1.0)


def test_logits_whose_values_are_not_side_by_side():
    # Every other value of wider rows: copied, and the gradient is the view's.
    z, v, idx, rest, y = _case((3, 6), 1003, 9, torch.bfloat16, 2.0, _gen(43))
    wide = torch.randn(3, 6, 2006, device="cuda").bfloat16()
    wide[..., ::2] = z
    view = wide[..., ::2]
    assert view.stride(-1) == 2 and not _twice(idx)
    for r, t, w in ((rest, y, 0.5), (None, None, 1.0)):
        _check_loss(view, v, idx, r, t, 2.0, w, w)
    # and with indices that are there twice, as halved ones are
    half = idx // 2
    assert _twice(half)
    _check_loss(view, v, half, rest, y, 2.0, 1.0, "twice")
