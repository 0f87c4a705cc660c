"""GPU tests of the embedding kernels (kernels/hip/embedding.py): the lookup with a scale and its gradient by sorted tokens."""

from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _tokens(how: str, M: int, V: int, g) -> torch.Tensor:
    u = torch.rand(M, generator=g, dtype=torch.float64, device="cuda")
    ids = {"uniform": lambda: (u * V).long(), "zipf": lambda: ((V + 1) ** u).long() - 1, "one": lambda: torch.full((M,), V // 2, device="cuda"),
           "two": lambda: torch.where(u < 0.5, 0, V - 1), "sorted": lambda: (u * V).long().sort().values}[how]()
    return ids.clamp_(0, V - 1)


def _scatter64(dy, idx, V):
    return torch.zeros(V, dy.shape[-1], dtype=torch.float64, device="cuda").index_add_(0, idx.reshape(-1), dy.double().reshape(-1, dy.shape[-1]))


# Lengths around a wave, a sort step (1024), a chunk's growth (16 at 32769, 32 at 65537 tokens) and a sort block of two
# steps (131073); vocabularies of one, two and three sorting passes (512 keys with the one of tokens that take no part);
# widths around the vectors and a wave's columns. Small whole numbers: every sum is exact, in any order.
@pytest.mark.parametrize("how", ["uniform", "zipf", "one", "two", "sorted"])
@pytest.mark.parametrize("M, V, N", [(1, 1, 1), (2, 3, 4), (7, 511, 8), (8, 512, 203), (9, 513, 260), (63, 1003, 64), (64, 5, 256), (65, 50304, 768), (1023, 7, 65),
                                     (1024, 50304, 32), (1025, 300000, 12), (8192, 50304, 96), (32769, 1003, 8), (70001, 50304, 4), (131073, 1003, 5)])
def test_gradient_of_whole_numbers_is_exact(M, V, N, how):
    from nanonemo_amd.kernels.hip import host

    print(f"\n[case] embedding gradient M={M} V={V} N={N} {how}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(M + V + N)
    idx = _tokens(how, M, V, g)
    dy = torch.randint(-4, 5, (M, N), generator=g, device="cuda").float()
    assert torch.equal(host().embedding_bwd(dy, idx, V, 1.0, -1).double(), _scatter64(dy, idx, V))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, T, V, N, how", [(1, 1, 50304, 768, "uniform"), (3, 37, 128, 96, "zipf"), (5, 777, 1003, 203, "zipf"), (8, 1024, 50304, 768, "zipf"), (2, 4096, 512, 1000, "one")])
def test_embedding_and_gradient_match_float64(B, T, V, N, how, dtype):
    from nanonemo_amd.kernels.hip.embedding import embedding

    print(f"\n[case] embedding B={B} T={T} V={V} N={N} {how} {dtype}", flush=True)
    g = torch.Generator(device="cuda").manual_seed(V + T)
    w = torch.randn(V, N, generator=g, device="cuda").to(dtype).requires_grad_()
    idx, scale = _tokens(how, B * T, V, g).view(B, T), float(torch.tensor(N**0.5))  # (a scale that fp32 holds)
    dy = torch.randn(B, T, N, generator=g, device="cuda").to(dtype)
    out = embedding(idx, w, scale)
    (dw,) = torch.autograd.grad(out, w, dy)
    assert out.dtype == dw.dtype == dtype and out.shape == (B, T, N) and dw.shape == w.shape
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    ref = w.detach().double()[idx] * scale
    # the fp32 product, and its rounding
    assert ((out.double() - ref).abs() <= (half + 2**-24) * (1 + half) * ref.abs() + tiny).all()
    ref = _scatter64(dy, idx, V) * scale
    # a sum of n values is a chain of at most 64 additions in a chunk, n / 64 over the chunks and 8 at the join
    n = min(B * T, 64 + B * T // 64 + 9)
    slack = (n + 1) * 2**-24 * _scatter64(dy.abs(), idx, V) * scale
    assert ((dw.double() - ref).abs() <= slack + half * (ref.abs() + slack) + tiny).all()
    assert torch.equal(dw, torch.autograd.grad(embedding(idx, w, scale), w, dy)[0])  # the same bits again


@pytest.mark.parametrize("dtype", DTYPES)
def test_unscaled_lookup_is_exact_and_keeps_special_values(dtype):
    from nanonemo_amd.kernels.hip.embedding import embedding

    for N in (1, 7, 64, 203):
        w = torch.randn(50, N, device="cuda").to(dtype)
        w[3] = float("inf")
        w[4] = -float("inf")
        w[5] = float("nan")
        w[6] = torch.finfo(dtype).max
        w[7] = torch.finfo(dtype).smallest_normal
        idx = torch.randint(0, 50, (3, 41), device="cuda")
        idx[0, :8] = torch.arange(8, device="cuda")
        torch.testing.assert_close(embedding(idx, w), F.embedding(idx, w), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("N", [64, 203])
def test_padding_and_tokens_out_of_range_take_no_part(N):
    from nanonemo_amd.kernels.hip.embedding import embedding

    g = torch.Generator(device="cuda").manual_seed(N)
    V = 37
    w = torch.randn(V, N, generator=g, device="cuda", requires_grad=True)
    idx = torch.randint(0, V, (4, 100), generator=g, device="cuda")
    idx[:, 80:] = 5
    dy = torch.randint(-4, 5, (4, 100, N), generator=g, device="cuda").float()
    dy[:, 80:] = float("nan")  # what a padded position's gradient holds does not matter
    for pad in (5, 5 - V):
        (dw,) = torch.autograd.grad(embedding(idx, w, padding_idx=pad), w, dy)
        ref = _scatter64(dy.nan_to_num(0.0), idx, V)
        ref[5] = 0
        assert torch.equal(dw.double(), ref)
    bad = idx.clone()
    bad[0, 3], bad[1, 4], bad[2, 5] = -1, V, 1 << 40
    out = embedding(bad, w)
    valid = (bad >= 0) & (bad < V)
    assert out[~valid].isnan().all() and torch.equal(out[valid], w[bad[valid]])
    (dw,) = torch.autograd.grad(out, w, dy.nan_to_num(1.0))
    assert torch.equal(dw.double(), _scatter64(dy.nan_to_num(1.0)[valid], bad[valid], V))
    none = torch.full((9,), V, device="cuda")  # no token takes part
    assert (torch.autograd.grad(embedding(none, w), w, dy[0, :9])[0] == 0).all()


def test_shapes_strides_and_types_of_the_inputs():
    from nanonemo_amd.kernels.hip.embedding import embedding

    w = torch.randn(203, 96, device="cuda", requires_grad=True)
    base = torch.randint(0, 203, (12, 10), device="cuda")
    big = torch.randn(12, 10, 192, device="cuda")
    for idx in (base, base.int(), base.t(), base[::2, 1:], base[0, 0], base[:0], base.t().int()[3:]):
        dy = big[..., ::2][: idx.numel()].reshape(-1)[: idx.numel() * 96].view(*idx.shape, 96)
        out, ref = embedding(idx, w), F.embedding(idx, w)
        assert torch.equal(out, ref)
        torch.testing.assert_close(torch.autograd.grad(out, w, dy)[0], torch.autograd.grad(ref, w, dy)[0], rtol=1e-5, atol=1e-5)
    out = embedding(base, w)
    expanded = torch.ones(1, 1, 1, device="cuda").expand(12, 10, 96)  # as sum() sends back
    assert torch.equal(torch.autograd.grad(out, w, expanded)[0].double(), _scatter64(expanded, base, 203))
    strided = big[..., ::2]
    assert torch.equal(torch.autograd.grad(embedding(base, w), w, strided)[0], torch.autograd.grad(embedding(base, w), w, strided.contiguous())[0])
    # a weight that starts anywhere, and one that is a transposed view
    flat = torch.randn(1 + 203 * 96, device="cuda")
    for v in (flat[1:].view(203, 96), torch.randn(96, 203, device="cuda").t()):
        assert torch.equal(embedding(base, v), v[base])


def test_op_and_eager_path_give_the_same_bits_and_the_op_passes_opcheck():
    from nanonemo_amd.kernels.hip.embedding import embedding

    idx = torch.randint(0, 203, (3, 50), device="cuda")
    w = torch.randn(203, 96, device="cuda", requires_grad=True)
    dy = torch.randn(3, 50, 96, device="cuda")
    out, op = embedding(idx, w, 1.5, 7), torch.ops.nanonemo.embedding(idx, w, 1.5, 7)
    assert 'EmbeddingNode' in out.grad_fn.name() and torch.equal(out, op)
    assert torch.equal(torch.autograd.grad(out, w, dy)[0], torch.autograd.grad(op, w, dy)[0])
    torch.library.opcheck(torch.ops.nanonemo.embedding, (idx, w, 1.5, 7))
    torch.library.opcheck(torch.ops.nanonemo.embedding_bwd, (dy, idx, 203, 1.5, 7))
    f = torch.compile(lambda i, t: embedding(i, t, 1.5, 7) * 2, fullgraph=True, backend="aot_eager")
    got = f(idx, w)
    assert torch.equal(got, op * 2)
    assert torch.equal(torch.autograd.grad(got, w, dy)[0], torch.autograd.grad(embedding(idx, w, 1.5, 7) * 2, w, dy)[0])
    with torch.no_grad():
        assert torch.equal(embedding(idx, w, 1.5, 7), out)


def test_the_autograd_node_refuses_what_it_cannot_do():
    from nanonemo_amd.kernels.hip.embedding import embedding

    idx = torch.randint(0, 20, (3, 5), device="cuda")
    w = torch.randn(20, 8, device="cuda", requires_grad=True)
    out = embedding(idx, w)
    (g,) = torch.autograd.grad(out.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    with pytest.raises(RuntimeError, match="batched gradients"):
        torch.autograd.grad(embedding(idx, w), w, torch.ones(2, 3, 5, 8, device="cuda"), is_grads_batched=True)
    out = embedding(idx, w)
    idx.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    out = embedding(idx, w)  # twice over one graph, and a hook on the way
    seen = []
    out.register_hook(lambda d: seen.append(d.shape))
    a, b = (torch.autograd.grad(out.sum(), w, retain_graph=True)[0] for _ in range(2))
    assert torch.equal(a, b) and len(seen) == 2
    loss = embedding(idx, w).sum()
    del out
    loss.backward()
    assert torch.equal(w.grad, a)


def test_on_another_stream_and_captured_into_a_graph():
    from nanonemo_amd.kernels.hip import host
    from nanonemo_amd.kernels.hip.embedding import embedding

    print("\n[case] embedding on a side stream and in a graph", flush=True)
    idx = torch.randint(0, 1003, (8, 300), device="cuda")
    w, dy = torch.randn(1003, 256, device="cuda"), torch.randn(8, 300, 256, device="cuda")
    ref, ref_dw = embedding(idx, w, 2.0), host().embedding_bwd(dy, idx, 1003, 2.0, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, dw = embedding(idx, w, 2.0), host().embedding_bwd(dy, idx, 1003, 2.0, 5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, ref) and torch.equal(dw, ref_dw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, dw = embedding(idx, w, 2.0), host().embedding_bwd(dy, idx, 1003, 2.0, 5)
    for i in range(4):
        new = torch.randint(0, 1003, idx.shape, device="cuda")
        dy.copy_(torch.randn_like(dy))
        idx.copy_(new)
        out.fill_(float("nan")), dw.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, embedding(idx, w, 2.0)) and torch.equal(dw, host().embedding_bwd(dy, idx, 1003, 2.0, 5)), i


@pytest.mark.parametrize("scale", [1.0, 16.0])
def test_model_with_the_embedding_kernel_matches_the_plain_one(scale):
    from nanonemo_amd.model import ModelConfig, NanoNemo

    small = dict(n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, d_ff=512, vocab_size=512, max_seq_len=128, emb_scale=scale, attn_kernel="hip_bthd", rope_kernel="hip", norm_kernel="hip")
    models, out = [], []
    for kernel in ("torch", "hip"):
        torch.manual_seed(0)
        models.append(NanoNemo(ModelConfig(**small, emb_kernel=kernel)).cuda())
    idx = torch.randint(0, 512, (2, 128), device="cuda")
    for m in models:
        with torch.autocast("cuda", dtype=torch.bfloat16):
            _, loss = m(idx, idx.roll(-1, 1))
        loss.backward()
        out.append((loss, {n: p.grad for n, p in m.named_parameters()}))
    assert list(models[0].state_dict()) == list(models[1].state_dict())
    assert torch.equal(out[0][0], out[1][0])  # the same values enter the first block
    for n, g in out[0][1].items():
        if n == "tok_emb.weight":  # another order of the same fp32 sums
            torch.testing.assert_close(out[1][1][n], g, rtol=1e-5, atol=1e-6 * g.abs().max().item())
        else:
            assert torch.equal(out[1][1][n], g), n


def test_refusals():
    from nanonemo_amd.kernels.hip import host
    from nanonemo_amd.kernels.hip.embedding import embedding

    w, idx = torch.randn(10, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for call, msg in ((lambda: embedding(idx.float(), w), "int64 or int32"), (lambda: embedding(idx, w.double()), "float32 matrix"), (lambda: embedding(idx, w[0]), "matrix|index"),
                      (lambda: embedding(idx.cpu(), w), "same device|CUDA"), (lambda: host().embedding_bwd(w[:2], idx, 10, 1.0, -1), "tokens' shape"),
                      (lambda: host().embedding_bwd(w[:3], idx, 10, 1.0, 10), "padding_idx"), (lambda: host().embedding_bwd(w[:3], idx, 0, 1.0, -1), "invalid sizes")):
        with pytest.raises((RuntimeError, IndexError), match=msg):
            call()


def test_the_module_keeps_pytorchs_lookup_for_what_the_kernels_do_not_take():
    from nanonemo_amd.model import Embedding

    idx = torch.randint(0, 50, (3, 7), device="cuda")
    for options, dtype in ((dict(), torch.float64), (dict(max_norm=1.0), torch.float32), (dict(scale_grad_by_freq=True), torch.float32)):
        m = Embedding(50, 16, 3.0, "hip", padding_idx=4, **options).cuda().to(dtype)
        ref = F.embedding(idx, m.weight, 4, **options) * 3.0
        out = m(idx)
        assert out.dtype == dtype and torch.equal(out, ref)
        assert torch.equal(torch.autograd.grad(out.sum(), m.weight)[0], torch.autograd.grad(ref.sum(), m.weight)[0])
    m = Embedding(50, 16, 3.0, "hip").cuda()
    assert "EmbeddingNode" in m(idx).grad_fn.name() and torch.equal(torch.jit.script(m)(idx), F.embedding(idx, m.weight) * 3.0)


def test_the_module_under_torch_funcs_transforms():
    from nanonemo_amd.model import Embedding

    m = Embedding(50, 16, 3.0, "hip", padding_idx=4).cuda()
    idx = torch.randint(0, 50, (3, 7), device="cuda")
    ref = torch.autograd.grad((F.embedding(idx, m.weight, 4) * 3.0).square().sum(), m.weight)[0]
    got = torch.func.grad(lambda t: torch.func.functional_call(m, {"weight": t}, (idx,)).square().sum())(m.weight.detach())
    assert torch.allclose(got, ref, rtol=21 * 2**-23, atol=0)  # (a sum of at most 21 equal terms, on either side)
    ws = torch.stack([m.weight.detach(), 2 * m.weight.detach()])
    both = torch.func.vmap(lambda t: torch.func.functional_call(m, {"weight": t}, (idx,)))(ws)
    assert torch.equal(both, torch.stack([F.embedding(idx, t) * 3.0 for t in ws]))
    assert torch.equal(torch.func.vmap(m)(idx), m(idx))
