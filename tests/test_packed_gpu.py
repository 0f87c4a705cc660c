"""GPU tests of attention over packed sequences (kernels/hip/packed.py): against float64, against the dense attention on each
sequence alone, bit for bit, and where it is called from."""

from __future__ import annotations

import math

import pytest
import torch

from tests.common import TOL, TOL_GRAD, assert_close_tol

pytestmark = pytest.mark.gpu

# lengths, H, KVH, hd: tile and unit edges with empty sequences; an odd group; one long sequence among short ones, whose pairs
# are split; few tokens, a block for each unit; many sequences, a wave for each pair; lengths of 1 and 2; long and split, MQA; short
# sequences alone, and many of them beside a longer one; a wave for each pair again, of single units that leave waves over and of
# pairs; a long one split at head_dim 32; long pairs that are not.
CASES = [
    ([63, 0, 64, 65, 1, 127, 128, 129, 0, 191, 192, 193, 0], 12, 4, 64),
    ([63, 64, 65, 1, 127, 128, 129, 300], 6, 2, 32),
    ([2500, 17, 130, 3], 12, 4, 64),
    ([200, 56], 12, 4, 64),
    ([100, 37, 64, 70] * 60, 12, 4, 64),
    ([1, 2, 1, 1, 3] * 80, 8, 8, 32),
    ([3000], 12, 1, 64),
    ([1111, 999, 1], 4, 4, 32),
    ([1, 31, 32, 33, 63, 64, 0, 2, 50] * 3, 12, 4, 64),
    ([40, 7, 64, 32, 5], 5, 1, 32),
    ([20, 64, 33] * 40 + [500], 8, 2, 64),
    ([100] * 343, 9, 3, 64),
    ([190, 129] * 130, 4, 4, 32),
    ([3000], 12, 1, 32),
    ([2100, 300], 32, 32, 64),
]
IDS = [f"{len(c[0])}x{max(c[0])}-{c[1]}-{c[2]}-{c[3]}" for c in CASES]


# What each case is there for: short tiles, splits, waves per pair (0: no longer sequences).
KINDS = [(0, 0, 4), (0, 0, 4), (0, 1, 4), (0, 0, 4), (1, 0, 4), (1, 0, None), (0, 1, 4), (0, 0, 4), (1, 0, None), (1, 0, None), (1, 0, 4), (0, 0, 1), (0, 0, 1), (0, 1, 4), (0, 0, 4)]


def _packing(lengths, H, KVH):
    from nanonemo_amd.kernels.hip.packed import Packing

    return Packing(lengths, H, KVH)


def _call(*args):
    from nanonemo_amd.kernels.hip.packed import flash_attn_packed

    return flash_attn_packed(*args)


def test_the_cases_are_of_every_kind():
    for (lengths, H, KVH, _), (few, split, wpp) in zip(CASES, KINDS):
        w = _packing(lengths, H, KVH).plan_host
        assert (w[16] > 0, w[10] > 0) == (few, split) and (wpp is None or w[11] == wpp), (lengths[:3], H, KVH, w[:18])
    single = [_packing(c[0], c[1], c[2]).plan_host for c in (CASES[3], CASES[14])]
    paired = [bool(w[w[13] + 7]) for w in single]
    assert paired == [False, True]


def _inputs(lengths, H, KVH, D, dtype, seed=0, mult=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(lengths)
    q, k, v = ((mult * torch.randn(T, n, D, device="cuda", generator=g)).to(dtype) for n in (H, KVH, KVH))
    return q, k, v, torch.randn(T, H, D, device="cuda", generator=g).to(dtype)


def _float64(q, k, v, do, lengths, between=None):
    """(o, dq, dk, dv) of the definition, a sequence and a head at a time, with dS rounded to a type between."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    group, scale, a = q.shape[1] // k.shape[1], 1 / math.sqrt(q.shape[2]), 0
    for n in lengths:
        r = slice(a, a + n)
        a += n
        future = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
        for h in range(q.shape[1] if n else 0):
            j = h // group
            p = torch.softmax((q[r, h] @ k[r, j].t() * scale).masked_fill(future, -math.inf), -1)
            o[r, h] = p @ v[r, j]
            dp = do[r, h] @ v[r, j].t()
            ds = p * (dp - (do[r, h] * o[r, h]).sum(-1, keepdim=True))
            ds = (ds if between is None else ds.to(between).double()) * scale
            dq[r, h] = ds @ k[r, j]
            dk[r, j] += ds.t() @ q[r, h]
            dv[r, j] += p.t() @ do[r, h]
    return o, dq, dk, dv


def _run(q, k, v, do, packing):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = _call(*leaves, packing)
    return (o.detach(), *torch.autograd.grad(o, leaves, do))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths, H, KVH, D", CASES, ids=IDS)
def test_matches_float64(lengths, H, KVH, D, dtype):
    print(f"\n[case] packed {len(lengths)} sequences of up to {max(lengths)}, H={H} KVH={KVH} D={D} {dtype}", flush=True)
    q, k, v, do = _inputs(lengths, H, KVH, D, dtype)
    got = _run(q, k, v, do, _packing(lengths, H, KVH))
    for name, x, ref, tol in zip(("o", "dq", "dk", "dv"), got, _float64(q, k, v, do, lengths), (TOL, TOL_GRAD, TOL_GRAD, TOL_GRAD)):
        assert_close_tol(x, ref, tol[dtype], name)


@pytest.mark.parametrize("lengths, H, KVH, D", CASES, ids=IDS)
def test_a_sequence_is_the_dense_attention_on_it_alone(lengths, H, KVH, D):
    from nanonemo_amd.kernels.hip import host
    from nanonemo_amd.kernels.hip.flash_attn import flash_attn_bthd

    print(f"\n[case] packed against dense, {len(lengths)} sequences of up to {max(lengths)}, H={H} KVH={KVH} D={D}", flush=True)
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=1)
    packing = _packing(lengths, H, KVH)
    plan = (packing.plan, packing.plan_host)
    o, lse, rest = host().packed_fwd(q, k, v, *plan, True)
    assert torch.equal(o, _call(q, k, v, packing))
    # without what rounding o left, as in the dense backward (but for sequences of one tile, below); with it dq is the same to its
    # rounding and dS's and D's (3 half steps)
    dq, dk, dv = host().packed_bwd(do, q, k, v, o, lse, rest.new_empty(0), *plan)
    for x, y in zip(host().packed_bwd(do, q, k, v, o, lse, rest, *plan), (dq, dk, dv)):
        assert (x.float() - y.float()).norm() <= 3 * 2**-9 * y.float().norm() + 1e-4
    a = 0
    for n in lengths[:20]:
        if n:
            alone = [t[None, a : a + n].clone().requires_grad_() for t in (q, k, v)]
            y = flash_attn_bthd(*alone)
            gq, gk, gv = torch.autograd.grad(y, alone, do[None, a : a + n].contiguous())
            assert torch.equal(y[0], o[a : a + n]), (a, n)
            if n <= 32 and packing.plan_host[16] > 0:  # (one tile: p is normalised again, and D comes of it and dp, not of o)
                # the dense dq and dk carry p's rounding in its sum and in o's D; either dS's and its own (dv: p's and its own): 2-norms
                # of 2^-8 (half steps) each, which add up in squares
                for x, y in ((gq[0], dq[a : a + n]), (gk[0], dk[a : a + n]), (gv[0], dv[a : a + n])):
                    assert (x.float() - y.float()).norm() <= math.sqrt(6) * 2**-8 * max(x.float().norm(), do[a : a + n].float().norm() * 2**-6), (a, n)
            else:
                assert torch.equal(gq[0], dq[a : a + n]), (a, n)
                # (dk and dv: other blocks may share the sums, each rounded to bf16 at the end: two roundings apart, and the fp32 sums' order)
                for x, y in ((gk[0], dk[a : a + n]), (gv[0], dv[a : a + n])):
                    torch.testing.assert_close(x.float(), y.float(), rtol=2**-7, atol=1e-5 * x.abs().max().item())
        a += n


def test_two_runs_give_the_same_bits():
    for lengths, H, KVH, D in (CASES[2], CASES[4], CASES[10]):
        q, k, v, do = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=2)
        packing = _packing(lengths, H, KVH)
        first = _run(q, k, v, do, packing)
        for again in (packing, _packing(torch.tensor(lengths), H, KVH)):
            assert all(torch.equal(a, b) for a, b in zip(first, _run(q, k, v, do, again)))


@pytest.mark.parametrize("lengths, H, KVH, D", [CASES[0], CASES[2], CASES[4], CASES[8], CASES[10]], ids=[IDS[0], IDS[2], IDS[4], IDS[8], IDS[10]])
def test_sequences_do_not_see_each_other(lengths, H, KVH, D):
    print(f"\n[case] packed among NaN, {len(lengths)} sequences", flush=True)
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=3)
    packing = _packing(lengths, H, KVH)
    ref = _run(q, k, v, do, packing)
    for parity in (0, 1):  # every other sequence of NaN and infinity
        bad = torch.cat([torch.full((n,), i % 2 == parity, device="cuda") for i, n in enumerate(lengths)])
        q2, k2, v2, do2 = (t.clone() for t in (q, k, v, do))
        for t, x in ((q2, math.nan), (k2, math.inf), (v2, math.nan), (do2, -math.inf)):
            t[bad] = x
        for a, b in zip(_run(q2, k2, v2, do2, packing), ref):
            assert torch.equal(a[~bad], b[~bad])


def test_rows_of_equal_and_of_large_scores():
    lengths, H, KVH, D = [300, 77, 1], 4, 2, 64
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=4)
    packing = _packing(lengths, H, KVH)
    o = _call(torch.zeros_like(q), k, v, packing)  # the mean of the values so far
    a = 0
    for n in lengths:
        mean = v[a : a + n].double().cumsum(0) / torch.arange(1, n + 1, device="cuda").view(-1, 1, 1)
        assert_close_tol(o[a : a + n], mean.repeat_interleave(2, 1), TOL[torch.bfloat16], "mean")
        a += n
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=5, mult=3.0)
    for name, x, ref, tol in zip(("o", "dq", "dk", "dv"), _run(q, k, v, do, packing), _float64(q, k, v, do, lengths), (TOL, TOL_GRAD, TOL_GRAD, TOL_GRAD)):
        assert_close_tol(x, ref, tol[torch.bfloat16], name)


def test_gradients_match_differences():
    lengths, H, KVH, D = [5, 1, 9], 4, 2, 32
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.float16, seed=6)
    packing = _packing(lengths, H, KVH)
    _, *grads = _run(q, k, v, do, packing)
    g = torch.Generator(device="cuda").manual_seed(7)
    for i, grad in enumerate(grads):
        # Along a direction of 0.25 steps, which fp16 holds beside values of up to 4 but for their own rounding (taken from what
        # the call is given). The loss is a sum of 15 * 4 * 32 products of outputs rounded to 11 bits: an error of 2^-11 of
        # about 1 each, of random sign: 2^-11 sqrt(1920) = 0.02 a side, over 2 * 0.25; third derivatives 0.25^2 / 6 of the
        # same order as the derivative.
        step = 0.25 * torch.sign(torch.randn(grad.shape, device="cuda", generator=g))
        ends = []
        for sign in (1, -1):
            ins = [q, k, v]
            ins[i] = (ins[i] + sign * step).half()
            ends.append((ins[i], (_call(*ins, packing).double() * do.double()).sum()))
        moved = ends[0][0].double() - ends[1][0].double()
        want, got = (ends[0][1] - ends[1][1]).item(), (grad.double() * moved).sum().item()
        size = (grad.double() * moved).norm().item()  # random signs: the size of the sum that is compared
        assert abs(got - want) <= 0.1 + 0.5 * size, (i, got, want, size)


def test_projections_are_read_in_place_and_other_layouts_copied():
    lengths, H, KVH, D = [70, 1, 200, 33], 12, 4, 64
    T = sum(lengths)
    packing = _packing(lengths, H, KVH)
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=8)
    ref = _run(q, k, v, do, packing)
    qkv = torch.cat([t.view(T, -1) for t in (q, k, v)], 1)
    cols = [t.view(T, -1, D) for t in qkv.split([H * D, KVH * D, KVH * D], 1)]  # a projection's column ranges
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]  # heads outermost
    odd = [torch.cat([t.new_zeros(4), t.flatten()])[4:].view(t.shape) for t in (q, k, v)]  # 8 bytes off
    wide = [torch.stack([t, t], -1)[..., 0] for t in (q, k, v)]  # values not side by side
    mixed = [cols[0], k, cols[2]]
    for views in (cols, turned, odd, wide, mixed):
        assert all(torch.equal(a, b) for a, b in zip(_run(*views, do, packing), ref))
    for d in (do.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([do.new_zeros(1), do.flatten()])[1:].view(do.shape)):
        assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, d, packing), ref))
    one = do[:, :1, :1].expand(T, H, D)  # a gradient without memory of its own
    assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, one, packing), _run(q, k, v, one.contiguous(), packing)))
    leaf = qkv.clone().requires_grad_()
    qs, ks, vs = (t.view(T, -1, D) for t in leaf.split([H * D, KVH * D, KVH * D], 1))
    (g,) = torch.autograd.grad(_call(qs, ks, vs, packing), leaf, do)
    assert torch.equal(g, torch.cat([t.view(T, -1) for t in ref[1:]], 1))


def test_nothing_to_do():
    for lengths in ([], [0], [0, 0]):
        packing = _packing(lengths, 4, 2)
        q, k, v, do = _inputs(lengths, 4, 2, 64, torch.bfloat16)
        assert [t.shape[0] for t in _run(q, k, v, do, packing)] == [0] * 4 and packing.positions.numel() == 0


def test_op_and_eager_path_give_the_same_bits_and_the_op_passes_opcheck():
    lengths, H, KVH, D = [70, 1, 0, 200, 33], 4, 2, 32
    packing = _packing(lengths, H, KVH)
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.float16, seed=9)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    o = _call(*leaves, packing)
    op, lse, rest = torch.ops.nanonemo.flash_attn_packed(*leaves, packing.plan, packing.plan_host, True)
    assert "PackedNode" in o.grad_fn.name() and torch.equal(o, op) and lse.shape == (H, sum(lengths))
    ref = torch.autograd.grad(o, leaves, do, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(ref, torch.autograd.grad(op, leaves, do)))
    torch.library.opcheck(torch.ops.nanonemo.flash_attn_packed, (*leaves, packing.plan, packing.plan_host, True))
    torch.library.opcheck(torch.ops.nanonemo.flash_attn_packed, (*(t.detach() for t in leaves), packing.plan, packing.plan_host, False))
    torch.library.opcheck(torch.ops.nanonemo.flash_attn_packed_bwd, (do, *(t.detach() for t in leaves), op.detach(), lse.detach(), rest, packing.plan, packing.plan_host))
    f = torch.compile(lambda a, b, c: _call(a, b, c, packing) * 2, fullgraph=True, backend="aot_eager")
    got = f(*leaves)
    assert torch.equal(got, o * 2)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, do), torch.autograd.grad(o * 2, leaves, do)))
    with torch.no_grad():
        assert torch.equal(_call(*leaves, packing), o)


def test_the_autograd_node_refuses_what_it_cannot_do():
    lengths, H, KVH, D = [20, 5], 4, 2, 32
    packing = _packing(lengths, H, KVH)
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.float16, seed=10)
    q.requires_grad_()
    (g,) = torch.autograd.grad(_call(q, k, v, packing).float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    with pytest.raises(RuntimeError, match="batched gradients"):
        torch.autograd.grad(_call(q, k, v, packing), q, torch.ones(2, *q.shape, device="cuda", dtype=q.dtype), is_grads_batched=True)
    o = _call(q, k, v, packing)
    v.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    o = _call(q, k, v, packing)
    a, b = (torch.autograd.grad(o, q, do, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(a, b)


def test_refusals():
    packing = _packing([20, 5], 4, 2)
    q, k, v, _ = _inputs([20, 5], 4, 2, 32, torch.float16)
    for call, msg in ((lambda: _call(q[:24], k[:24], v[:24], packing), "the packing is of 25 tokens"), (lambda: _call(q[:, :2], k, v, packing), "the packing is of"), (lambda: _call(q, q, q, packing), "the packing is of"),
                      (lambda: _call(q.float(), k.float(), v.float(), packing), "float16 or bfloat16"), (lambda: _call(q, k, v[:, :1], packing), "expected"), (lambda: _call(q[None], k[None], v[None], packing), "expected"),
                      (lambda: _call(q[..., :16], k[..., :16], v[..., :16], packing), "head_dim"), (lambda: _call(q, k.cpu(), v, packing), "same device|CUDA"), (lambda: _call(q, k.bfloat16(), v, packing), "same dtype"),
                      (lambda: torch.ops.nanonemo.flash_attn_packed(q, k, v, packing.plan[:-1], packing.plan_host, False), "Packing's"),
                      (lambda: torch.ops.nanonemo.flash_attn_packed(q, k, v, packing.plan, packing.plan, False), "Packing's"),
                      (lambda: torch.ops.nanonemo.flash_attn_packed(q, k, v, torch.zeros_like(packing.plan), torch.zeros_like(packing.plan_host), False), "not a plan")):
        with pytest.raises(RuntimeError, match=msg):
            call()


def test_on_another_stream_and_captured_into_a_graph():
    from nanonemo_amd.kernels.hip import host

    print("\n[case] packed attention on a side stream and in a graph", flush=True)
    lengths, H, KVH, D = [1500, 70, 33], 12, 4, 64  # split: the partial sums' launch too
    packing = _packing(lengths, H, KVH)
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=11)

    def both():
        o, lse, rest = host().packed_fwd(q, k, v, packing.plan, packing.plan_host, True)
        return (o, *host().packed_bwd(do, q, k, v, o, lse, rest, packing.plan, packing.plan_host))

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
        for t in (q, k, v, do):
            t.copy_(torch.randn_like(t))
        for t in outs:
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, both())), i


SMALL = dict(n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, d_ff=512, vocab_size=512, max_seq_len=256, attn_backend="math_fp32")


def _step(cfg, state, idx, y, lengths):
    from nanonemo_amd.model import ModelConfig, NanoNemo

    model = NanoNemo(ModelConfig(**SMALL, **cfg)).cuda()
    model.load_state_dict(state)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits, loss = model(idx, y, None, model.pack(lengths) if lengths else None)
    loss.backward()
    return loss.item(), logits.float(), {n: p.grad for n, p in model.named_parameters()}


@pytest.mark.parametrize("qk_norm", [False, True])
@pytest.mark.parametrize("attn, rope", [("hip_bthd", "hip"), ("hip", "hip"), ("hip_bthd", "torch"), ("hip_bthd", "fused")])
@pytest.mark.parametrize("lengths", [None, [200, 1, 55, 0, 130, 126]])
def test_model_with_the_kernels_matches_the_plain_one(lengths, attn, rope, qk_norm):
    from nanonemo_amd.model import ModelConfig, NanoNemo

    if lengths is None and not qk_norm:
        pytest.skip("the dense model without the norm is tested elsewhere")
    print(f"\n[case] model attn={attn} rope={rope} qk_norm={qk_norm} lengths={lengths}", flush=True)
    torch.manual_seed(0)
    state = NanoNemo(ModelConfig(**SMALL, qk_norm=qk_norm)).state_dict()
    for n, t in state.items():
        if n.endswith(("q_norm.weight", "k_norm.weight")):
            t.normal_(1.0, 0.2)
    idx, y = (torch.randint(0, 512, (2, 256), device="cuda") for _ in range(2))
    y[0, 199] = -100
    plain = _step(dict(qk_norm=qk_norm), state, idx, y, lengths)
    got = _step(dict(qk_norm=qk_norm, attn_kernel=attn, rope_kernel=rope, norm_kernel="hip"), state, idx, y, lengths)
    # bf16 activations: 2^-8 for each of some ten roundings a block on values that the norms keep at 1, at random: 2^-8 sqrt(20),
    # times the output weights' 0.02 sqrt(256) = 0.32 for a logit; the loss averages 511 of them. Gradients: as the model's other
    # kernels are held to, a twentieth of the tensor's norm.
    assert abs(got[0] - plain[0]) < 5e-3
    assert (got[1] - plain[1]).abs().max() < 5 * 2**-8 * math.sqrt(20) * 0.32
    for n, g in plain[2].items():
        assert (got[2][n] - g).norm() <= 0.05 * g.norm() + 1e-6, n


def test_packed_training_step():
    from nanonemo_amd.model import ModelConfig, NanoNemo
    from nanonemo_amd.train import make_optimizer, packed_batches, synthetic_documents, teacher_batches, train_step

    torch.manual_seed(0)
    cfg = ModelConfig(**SMALL, attn_kernel="hip_bthd", rope_kernel="hip", norm_kernel="hip", emb_kernel="hip", qk_norm=True)
    model, teacher = NanoNemo(cfg).cuda(), NanoNemo(cfg).cuda()
    batches = packed_batches(model, synthetic_documents(2, 600, 70, 512), 600)
    assert len(batches) >= 2 and all(x.is_cuda and p.device.type == "cuda" for x, _, _, p in batches)
    before = {n: p.clone() for n, p in model.named_parameters()}
    opt = make_optimizer(model)
    for some in (batches[:2], teacher_batches(teacher, batches[:2], 8)):
        loss, norm = train_step(model, opt, some)
        assert loss.isfinite() and norm.isfinite()
    assert all(not torch.equal(before[n], p) for n, p in model.named_parameters())


def test_the_two_operators_together():
    """A model's attention between its projections: norm and rotation of q and k where they lie, attention within sequences, and
    the gradient of the projection and the norms' weights, against float64 with the roundings between the two counted."""
    from nanonemo_amd.kernels.hip.qk_norm import qk_norm_rope

    lengths, H, KVH, D = [130, 1, 0, 64, 45, 260], 12, 4, 64
    T = sum(lengths)
    packing = _packing(lengths, H, KVH)
    g = torch.Generator(device="cuda").manual_seed(12)
    qkv = (2 * torch.randn(T, (H + 2 * KVH) * D, device="cuda", generator=g)).bfloat16().requires_grad_()
    wq, wk = ((1 + 0.2 * torch.randn(D, device="cuda", generator=g)).requires_grad_() for _ in range(2))
    do = torch.randn(T, H, D, device="cuda", generator=g).bfloat16()
    angle = torch.outer(torch.arange(300, dtype=torch.float64), 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D))
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()

    def chain(qkv, wq, wk, cos, sin, rotate, attend):
        q, k, v = (t.view(T, -1, D) for t in qkv.split([H * D, KVH * D, KVH * D], 1))
        return attend(*rotate(q, k, wq, wk, cos, sin), v)

    o = chain(qkv, wq, wk, cos, sin, lambda *a: qk_norm_rope(*a, packing.positions), lambda *a: _call(*a, packing))
    got = (o.detach(), *torch.autograd.grad(o, (qkv, wq, wk), do))

    def rotate64(q, k, wq, wk, cos, sin):
        c, s = (t[packing.positions].unsqueeze(1) for t in (cos, sin))
        outs = []
        for x, w in ((q, wq), (k, wk)):
            a, b = (w * x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-5)).chunk(2, -1)
            outs.append(torch.cat((a * c - b * s, a * s + b * c), -1))
        return outs

    def attend64(q, k, v):
        outs = []
        for a, b, c in zip(q.split(lengths), k.split(lengths), v.split(lengths)):
            b, c = b.repeat_interleave(H // KVH, 1), c.repeat_interleave(H // KVH, 1)
            x = torch.matmul(a.transpose(0, 1), b.permute(1, 2, 0)) / math.sqrt(D)
            x = x.masked_fill(torch.ones(x.shape[1:], dtype=torch.bool, device="cuda").triu(1), -math.inf)
            outs.append(torch.matmul(x.softmax(-1), c.transpose(0, 1)).transpose(0, 1))
        return torch.cat(outs)

    ins = [t.detach().double().requires_grad_() for t in (qkv, wq, wk)]
    ref = chain(*ins, cos.double(), sin.double(), rotate64, attend64)
    want = (ref.detach(), *torch.autograd.grad(ref, ins, do.double()))
    # (q and k between the two are rounded to bf16: the errors of o and the gradients double at most in the norm, 2 * TOL's fro)
    for name, x, y, tol in zip(("o", "dqkv", "dwq", "dwk"), got, want, (TOL, TOL_GRAD, TOL_GRAD, TOL_GRAD)):
        assert_close_tol(x, y, {**tol[torch.bfloat16], "fro": 2 * tol[torch.bfloat16]["fro"]}, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_carry_two_roundings(dtype):
    """dS is rounded to 16 bits before its products and a gradient once more: errors of like size, independent, so sqrt(2) = 1.42
    of one rounding's. The bound of 1.5 leaves 6 % for lse, P and the fp32 sums; with a D from the rounded o it fails."""
    for lengths, H, KVH, D in (([1000, 300, 77], 4, 2, 64), ([64, 33, 50] * 30, 4, 2, 64), ([700, 90], 4, 4, 32)):
        q, k, v, do = _inputs(lengths, H, KVH, D, dtype, seed=13)
        _, *got = _run(q, k, v, do, _packing(lengths, H, KVH))
        for name, x, ref in zip(("dq", "dk"), got, _float64(q, k, v, do, lengths)[1:]):
            one = (ref.to(dtype).double() - ref).norm()
            ratio = ((x.double() - ref).norm() / one).item()
            print(f"[err] {name} {ratio:.3f} roundings", flush=True)
            assert ratio <= 1.5, (name, lengths[:3], ratio)


def test_packings_of_inference_mode_and_two_streams_at_once():
    lengths, H, KVH, D = [700, 30, 129], 12, 4, 64
    with torch.inference_mode():
        packing = _packing(lengths, H, KVH)
        q, k, v, do = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=14)
        inferred = _call(q, k, v, packing)
    ins = [t.clone() for t in (q, k, v, do)]
    ref = _run(*ins, packing)
    assert torch.equal(ref[0], inferred)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(4):
        for st in streams:  # the same packing on both, their workspaces their own
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                outs.append(_run(*ins, packing))
    for st in streams:
        torch.cuda.current_stream().wait_stream(st)
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, ref))


def test_packed_model_compiles_without_graph_breaks():
    from nanonemo_amd.model import ModelConfig, NanoNemo

    torch.manual_seed(0)
    model = NanoNemo(ModelConfig(**SMALL, attn_kernel="hip_bthd", rope_kernel="hip", norm_kernel="hip", qk_norm=True)).cuda()
    lengths = [100, 28, 1, 127]
    packing = model.pack(lengths)
    idx, y = (torch.randint(0, 512, (1, 256), device="cuda") for _ in range(2))

    def loss(m):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return m(idx, y, None, packing)[1]

    got, want = loss(torch.compile(model, fullgraph=True, backend="aot_eager")), loss(model)
    # the compiled modules round weight gradients and the loss's logits as autocast does: bf16 logits of about 0.3 in both
    torch.testing.assert_close(got, want, rtol=2e-3, atol=0)
    got.backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in model.parameters())


def test_evaluation_of_a_packed_model_captured_into_a_graph():
    from nanonemo_amd.model import ModelConfig, NanoNemo

    print("\n[case] packed model in a graph", flush=True)
    torch.manual_seed(0)
    model = NanoNemo(ModelConfig(**SMALL, attn_kernel="hip_bthd", rope_kernel="hip", norm_kernel="hip", emb_kernel="hip", qk_norm=True)).cuda()
    packing = model.pack([100, 28, 1, 127])
    idx = torch.randint(0, 512, (1, 256), device="cuda")

    def run():
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            return model(idx, packing=packing)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for i in range(4):
        idx.copy_(torch.randint(0, 512, idx.shape, device="cuda"))
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run()), i


def test_offsets_past_32_bits():
    """The last sequence of 2.9 million tokens, whose values lie past the 2^31st of q, o and the gradients."""
    print("\n[case] 2.9 million packed tokens", flush=True)
    H, KVH, D = 12, 4, 64
    lengths = [1024] * 2800 + [20] * 30 + [300, 33]  # (many short ones, and a longer one behind them)
    T = sum(lengths)
    assert (T - 333) * H * D > 2**31
    last = 333
    tail = _inputs([300, 33], H, KVH, D, torch.bfloat16, seed=15)
    q, k, v, do = (torch.zeros(T, n, D, dtype=torch.bfloat16, device="cuda") for n in (H, KVH, KVH, H))
    for t, x in zip((q, k, v, do), tail):
        t[-last:] = x
    got = _run(q, k, v, do, _packing(lengths, H, KVH))
    small = _packing([300, 33], H, KVH)
    for name, x, y in zip(("o", "dq", "dk", "dv"), got, _run(*tail, small)):
        assert not x[:-last].any(), name
        # (which blocks share a sum goes by the batch: fp32 sums in another order, rounded to bf16)
        torch.testing.assert_close(x[-last:].float(), y.float(), rtol=2**-7, atol=1e-5 * y.float().abs().max().item(), msg=name)
    assert torch.equal(got[0][-last:], _call(*tail[:3], small))


# (whole blocks, short ones, a wave a pair beside short ones, shared pairs)
@pytest.mark.parametrize("lengths", [[300, 1000, 5], [30] * 40, [700] * 60 + [20] * 400, [4096]])
def test_a_list_that_was_overwritten_costs_values_only(lengths):
    """A program that frees a packing while a captured graph or another stream still reads it: entries that lie outside the
    tensors are passed over, and what else the memory holds stays as it was."""
    print(f"\n[case] overwritten list of {len(lengths)} sequences", flush=True)
    H, KVH, D = 12, 4, 64
    q, k, v, do = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=12)
    packing = _packing(lengths, H, KVH)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    want = _run(q, k, v, do, packing)
    mine = packing.plan.clone()
    g = torch.Generator().manual_seed(13)
    T = sum(lengths)
    for low, high in ((2**31 - 1, 2**31), (-1, 0), (0, 1), (-(2**31), 2**31), (-2, T + 3), (-1, 40), (0, 4)):
        packing.plan.copy_(torch.randint(low, high, mine.shape, generator=g).to(torch.int32))
        o = _call(*leaves, packing)
        torch.autograd.grad(o, leaves, do)
        torch.cuda.synchronize()
        for a, b in zip(leaves, (q, k, v)):
            assert torch.equal(a.detach(), b)
    packing.plan.copy_(mine)
    for a, b in zip(_run(q, k, v, do, packing), want):
        assert torch.equal(a, b)


LAYER = [([100, 1, 260, 0, 64, 33], 12, 4, 64), ([20] * 30, 2, 2, 64), ([700, 330], 8, 2, 32), ([130, 1, 65], 4, 1, 32)]


def _layer(lengths, H, KVH, hd):
    """An attention layer, its packing, and cos and sin of every token."""
    from tests.test_layers_gpu import _attention

    m, (cos, sin) = _attention(H, KVH, hd, max(lengths), rope_kernel="hip")
    packing = _packing(lengths, H, KVH)
    return m, packing, cos[packing.positions], sin[packing.positions]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths, H, KVH, hd", LAYER)
def test_packed_attention_layer_matches_its_modules_and_float64(lengths, H, KVH, hd, dtype):
    from tests.test_layers_gpu import _assert_close_to_float64, _attention64, _modules_only
    from tests.test_layers_gpu import _run as run

    print(f"\n[case] packed attention layer of {len(lengths)} sequences H={H} KVH={KVH} hd={hd} {dtype}", flush=True)
    m, packing, cos, sin = _layer(lengths, H, KVH, hd)
    T = sum(lengths)
    x = torch.randn(1, T, H * hd, device="cuda").to(dtype).requires_grad_()
    dy = torch.randn(1, T, H * hd, device="cuda").to(dtype)
    got, ref = run(m, (x, cos, sin, packing), dy, dtype), run(_modules_only(m), (x, cos, sin, packing), dy, dtype)
    ins = [t.detach().double().requires_grad_() for t in (x, m.wq.weight, m.wk.weight, m.wv.weight, m.wo.weight)]
    # (the rows of each sequence's own tables are the first of the longest one's)
    i = lengths.index(max(lengths))
    a = sum(lengths[:i])
    c, s = cos[a : a + lengths[i]], sin[a : a + lengths[i]]
    y = torch.cat([_attention64(t, c, s, H, KVH, *ins[1:]) for t in ins[0].split(lengths, 1) if t.shape[1]], 1)
    exact = (y.detach(), *torch.autograd.grad(y, ins, dy.double()))
    # as the dense layer: weights, product, rotation of q and of k; P and O; the output weight, dO, dS, dq or dk, its rotation
    _assert_close_to_float64(("y", "dx", "dwq", "dwk", "dwv", "dwo"), got, ref, exact, 13, dtype)
    with torch.no_grad(), torch.autocast("cuda", dtype=dtype):
        assert torch.equal(m(x, cos, sin, packing), got[0])


def test_packed_attention_layer_is_one_node():
    m, packing, cos, sin = _layer([70, 70], 4, 2, 64)
    x = torch.randn(1, 140, 256, device="cuda", requires_grad=True)  # fp32 in, cast by the layer
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x, cos, sin, packing)
    node = y.grad_fn
    while "View" in node.name():
        node = node.next_functions[0][0]
    assert node.name() == "_AttentionLayerBackward"


def test_packed_attention_layer_frozen_parts_and_repeated_backward():
    m, packing, cos, sin = _layer([70, 30, 40], 4, 2, 64)
    x = torch.randn(1, 140, 256, device="cuda", requires_grad=True)
    m.wk.weight.requires_grad_(False)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x, cos, sin, packing)
    y.float().square().sum().backward(retain_graph=True)
    first = [t.grad.clone() for t in (x, m.wq.weight, m.wv.weight, m.wo.weight)]
    assert m.wk.weight.grad is None
    y.float().square().sum().backward()
    for a, t in zip(first, (x, m.wq.weight, m.wv.weight, m.wo.weight)):
        assert torch.equal(a + a, t.grad)
    for p in m.parameters():
        p.requires_grad_(False)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        (gx,) = torch.autograd.grad(m(x, cos, sin, packing).float().square().sum(), x)
    assert torch.equal(gx, first[0])
    m.wo.weight.requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        (gw,) = torch.autograd.grad(m(x.detach(), cos, sin, packing).float().square().sum(), m.wo.weight)
    assert torch.equal(gw, first[3])


def test_packed_attention_layer_recorded_and_batched_backwards():
    """They go through the modules' functions: first derivatives by the kernels, second and batched ones through the attention refused."""
    from tests.test_layers_gpu import _modules_only

    m, packing, cos, sin = _layer([20, 13], 4, 2, 32)
    x = torch.randn(1, 33, 128, device="cuda", requires_grad=True)
    out = []
    for mod in (m, _modules_only(m)):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = mod(x, cos, sin, packing)
        (gw,) = torch.autograd.grad(y.float().sum(), mod.wo.weight, create_graph=True)
        out.append(torch.autograd.grad(gw.square().sum(), x))
    for a, b in zip(*out):
        torch.testing.assert_close(a, b, rtol=5e-2, atol=5e-2 * b.abs().max().item())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x, cos, sin, packing)
    (gx,) = torch.autograd.grad(y.float().sum(), x, create_graph=True)
    # (as with PyTorch's own once_differentiable the graph of gx ends at the node that refuses: x is not in it, and a backward meets it)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        gx.square().sum().backward()
    with pytest.raises(RuntimeError, match="batched gradients"):
        torch.autograd.grad(y, x, torch.ones(2, *y.shape, device="cuda", dtype=y.dtype), is_grads_batched=True)


def test_packed_attention_layer_refuses_another_batch_s_packing():
    m, packing, cos, sin = _layer([20, 13], 4, 2, 32)
    x = torch.randn(1, 33, 128, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for bad in (_packing([20, 12], 4, 2), _packing([20, 13], 4, 4), _packing([20, 13], 2, 2)):
            with pytest.raises(RuntimeError, match="packing"):
                m(x, cos, sin, bad)


@pytest.mark.parametrize("what", ["layer", "flash_attn_packed", "qk_norm_rope"])
def test_saved_tensors_are_checked_like_inputs(what):
    """What a saved-tensor hook hands back reaches the kernels by address: dense or not it is read rightly, and a host tensor or
    another type is an error before any launch."""
    from nanonemo_amd.kernels.hip.qk_norm import qk_norm_rope
    from tests.test_layers_gpu import _rel, _saved_through

    m, packing, cos, sin = _layer([70, 30, 40], 4, 2, 64)
    x = torch.randn(1, 140, 256, device="cuda").bfloat16().requires_grad_()
    q, k, v = (torch.randn(140, h, 64, device="cuda").bfloat16().requires_grad_() for h in (4, 2, 2))
    wq, wk = (torch.ones(64, device="cuda", requires_grad=True) for _ in range(2))

    def f():
        if what == "layer":
            with torch.autocast("cuda", dtype=torch.bfloat16):
                return m(x, cos, sin, packing), (x, *m.parameters())
        if what == "flash_attn_packed":
            return _call(q, k, v, packing), (q, k, v)
        a, b = qk_norm_rope(q, k, wq, wk, cos, sin)
        return torch.cat((a, b), 1), (q, k, wq, wk)

    def spread(t):  # the same values, every second element of a buffer
        return t if t.dim() == 0 else torch.stack((t, t), -1)[..., 0]

    ref = _saved_through(lambda t: t, f)
    for a, b in zip(_saved_through(spread, f), ref):
        # (the library may take another product for other strides: two bf16 roundings apart)
        assert torch.equal(a, b) or what == "layer" and _rel(a, b.double()) < 2 * 2.0**-8
    for bad in (lambda t: t.cpu(), lambda t: t.float() if t.dtype == torch.bfloat16 else t):
        with pytest.raises(RuntimeError):
            _saved_through(bad, f)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("most", [2, 5, 12, 32])
def test_gradients_of_short_sequences_carry_two_roundings_alone(most, dtype):
    """Rows with few keys, where a D from rounded p would be as far off as dS's own rounding is: dq and dk are as near as float64
    with just the two roundings that the kernel makes, dS's for the products and its result's. (Their size goes by where values lie
    between powers of two, so the bound is what those two do to these values.)"""
    g = torch.Generator().manual_seed(most)
    lengths = torch.randint(1, most + 1, (800,), generator=g).tolist()
    H, KVH, D = 4, 2, 64
    q, k, v, do = _inputs(lengths, H, KVH, D, dtype, seed=most)
    got = _run(q, k, v, do, _packing(lengths, H, KVH))
    want = _float64(q, k, v, do, lengths)
    twice = _float64(q, k, v, do, lengths, between=dtype)
    for name, x, y, z in zip(("dq", "dk"), got[1:3], want[1:3], twice[1:3]):
        off, least, once = ((t.to(dtype).double() - y).norm() for t in (x, z, y))
        print(f"  {name} of sequences of up to {most}, {dtype}: {(off / once).item():.3f} roundings, two are {(least / once).item():.3f}", flush=True)
        # (values between two steps, which fp32's errors of some 2^-22 send the other way, are one in 2^13 or fewer)
        assert off <= 1.02 * least, name


def _shifted(t):
    """The same values one element into a buffer, off the 16-byte boundaries of which the kernels read."""
    return torch.cat([t.new_zeros(1), t.flatten()])[1:].view(t.shape)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("qk_norm", [False, True])
def test_attention_layer_takes_tables_off_a_boundary(qk_norm, packed):
    """As the norm's own call does: in the fused layer, in its recorded backward, module by module, and negated lazily."""
    from tests.test_layers_gpu import _attention, _modules_only

    print(f"\n[case] attention layer, tables off a boundary, qk_norm={qk_norm} packed={packed}", flush=True)
    lengths = [20, 13] if packed else None
    m, (cos, sin) = _attention(4, 2, 64, 33, rope_kernel="hip", qk_norm=qk_norm)
    more = ()
    if packed:
        more = (_packing(lengths, 4, 2),)
        cos, sin = cos[more[0].positions], sin[more[0].positions]
    x = torch.randn(1, 33, 256, device="cuda").bfloat16().requires_grad_()
    dy = torch.randn(1, 33, 256, device="cuda").bfloat16()

    def run(mod, c, s, **kw):
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = mod(x, c, s, *more)
        return (y.detach(), *(g.detach() for g in torch.autograd.grad(y, (x, *mod.parameters()), dy, **kw)))

    odd = [_shifted(t) for t in (cos, sin)]
    assert all(t.is_contiguous() and t.data_ptr() % 16 for t in odd)
    lazy = [torch._neg_view(-t) for t in (cos, sin)]
    assert all(t.is_neg() and t.is_contiguous() for t in lazy)
    for mod, kw in ((m, {}), (_modules_only(m), {}), (m, dict(create_graph=True))):
        want = run(mod, cos, sin, **kw)
        for tables in (odd, lazy):
            for a, b in zip(run(mod, *tables, **kw), want):
                assert torch.equal(a, b)


def test_rotations_take_tables_off_a_boundary():
    from nanonemo_amd.kernels.hip.flash_attn import flash_attn_bthd_rope
    from nanonemo_amd.kernels.hip.rope import rope_k, rope_qk
    from nanonemo_amd.model import rope_tables

    print("\n[case] rotations, tables off a boundary", flush=True)
    q, k, v = (torch.randn(2, 33, h, 64, device="cuda").bfloat16().requires_grad_() for h in (4, 2, 2))
    tables = [t.cuda() for t in rope_tables(64, 40, 10000.0)]
    for f in (lambda *t: torch.cat(rope_qk(q, k, *t), 2), lambda *t: rope_k(k, *t), lambda *t: flash_attn_bthd_rope(q, k, v, *t)):
        outs = []
        for t in (tables, [_shifted(t) for t in tables]):
            y = f(*t)
            outs.append((y.detach(), *torch.autograd.grad(y.float().square().sum(), (q, k, v), allow_unused=True)))
        for a, b in zip(*outs):
            assert a is None and b is None or torch.equal(a, b)


def test_the_layer_s_norms_come_back_from_saved_tensor_hooks_off_a_boundary():
    from tests.test_layers_gpu import _attention, _saved_through

    m, (cos, sin) = _attention(4, 2, 64, 33, rope_kernel="hip", qk_norm=True)
    x = torch.randn(1, 33, 256, device="cuda").bfloat16().requires_grad_()

    def f():
        with torch.autocast("cuda", dtype=torch.bfloat16):
            return m(x, cos, sin), (x, *m.parameters())

    ref = _saved_through(lambda t: t, f)
    for a, b in zip(_saved_through(lambda t: _shifted(t) if t.dim() == 1 and t.dtype == torch.float32 else t, f), ref):
        assert torch.equal(a, b)


@pytest.mark.parametrize("lengths", [[300, 1000, 5], [30] * 40 + [50] * 20, [700] * 60 + [20] * 400, [4096]])
def test_a_list_that_was_overwritten_leaves_the_memory_around_the_tensors(lengths):
    """What the kernels write lies side by side with rows of a pattern between: none of it changes, nor does what they read,
    whatever the list holds (random words; the list's own, some of them one off or another entry's)."""
    import ctypes

    from nanonemo_amd.kernels.hip import check, lib

    print(f"\n[case] overwritten list of {len(lengths)} sequences among guards", flush=True)
    H, KVH, D = 12, 4, 64
    ins = _inputs(lengths, H, KVH, D, torch.bfloat16, seed=16)
    packing = _packing(lengths, H, KVH)
    host, words, T, L = packing.plan_host.data_ptr(), len(packing.plan), sum(lengths), lib()
    ws = L.nn_fa_packed_bwd_workspace_size(host, D)
    q, kv = 2 * T * H * D, 2 * T * KVH * D
    names = ("q", "k", "v", "do", "plan", "o", "lse", "rest", "dq", "dk", "dv", "ws")
    sizes = dict(zip(names, (q, kv, kv, q, 4 * words, q, 4 * H * T, q // 2, q, kv, kv, ws)))
    guard, at, end = 1 << 16, {}, 1 << 16
    for n in names:
        at[n] = end
        end = (end + sizes[n] + guard + 255) // 256 * 256
    memory = torch.full((end,), 0x5A, dtype=torch.uint8, device="cuda")
    for n, t in zip(names, ins):
        memory[at[n] : at[n] + sizes[n]] = t.flatten().view(torch.uint8)
    # (everything but what the kernels may write, and the list)
    kept = torch.ones(end, dtype=torch.bool, device="cuda")
    for n in names[4:]:
        kept[at[n] : at[n] + sizes[n]] = False
    before = memory[kept]
    a = {n: memory.data_ptr() + at[n] for n in names}
    plan = memory[at["plan"] : at["plan"] + 4 * words].view(torch.int32)
    stream = torch.cuda.current_stream().cuda_stream

    def run():
        s = ctypes.c_float(D**-0.5)
        check(L.nn_fa_packed_fwd(a["q"], a["k"], a["v"], a["o"], a["lse"], a["rest"], host, a["plan"], D, None, 1, s, stream))
        check(L.nn_fa_packed_bwd(a["do"], a["q"], a["k"], a["v"], a["o"], a["lse"], a["rest"], a["dq"], a["dk"], a["dv"], a["ws"], ws, host, a["plan"],
                                 D, None, 1, s, stream))
        torch.cuda.synchronize()

    g = torch.Generator().manual_seed(17)
    mine = packing.plan_host
    lists = [torch.randint(low, high, mine.shape, generator=g).to(torch.int32)
             for low, high in ((2**31 - 1, 2**31), (-1, 0), (0, 1), (-(2**31), 2**31), (-2, T + 3), (-1, 40), (0, 4))]
    lists += [mine + torch.randint(-1, 2, mine.shape, generator=g, dtype=torch.int32) * (torch.rand(mine.shape, generator=g) < 0.2) for _ in range(4)]
    lists += [torch.where(torch.rand(mine.shape, generator=g) < 0.2, mine[torch.randperm(words, generator=g)], mine) for _ in range(4)]
    for i, bad in enumerate([*lists, mine]):
        plan.copy_(bad)
        run()
        assert torch.equal(memory[kept], before), i
        assert torch.equal(plan.cpu(), bad), i
    want = _run(*ins, packing)
    for n, t in zip(("o", "dq", "dk", "dv"), want):
        assert torch.equal(memory[at[n] : at[n] + sizes[n]].view(torch.bfloat16), t.flatten()), n
