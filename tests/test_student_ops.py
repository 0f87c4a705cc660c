"""CPU tests of the operators at the ends of a student's training step (embedding, top logits, distillation loss): schemas,
fake impls, argument checks at the C ABI and in the public functions, and the model's use of them. No GPU compute is launched
here."""

from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

from nanonemo_amd.kernels.hip import check_distill, check_embedding, lib
from nanonemo_amd.model import ModelConfig, NanoNemo, Teacher, distill_loss
from nanonemo_amd.train import make_optimizer, teacher_batches, train_step

SMALL = dict(n_layers=1, d_model=64, n_heads=2, n_kv_heads=1, d_ff=64, vocab_size=96, max_seq_len=16)


@pytest.mark.parametrize(
    "kw, msg",
    [
        (dict(M=-1), "invalid sizes"),
        (dict(M=1 << 31), "invalid sizes"),
        (dict(V=0), "invalid sizes"),
        (dict(V=1 << 27), "invalid sizes"),
        (dict(N=0), "invalid sizes"),
        (dict(N=1 << 20), "invalid sizes"),
        (dict(dtype=3), "dtype must be float16, bfloat16 or float32"),
        (dict(bits=16), "tokens must be int32 or int64"),
        (dict(w=24), "16-byte aligned"),
        (dict(w=None), "null pointer"),
        (dict(idx=None), "null pointer"),
    ],
)
def test_embedding_c_abi_rejects_bad_arguments_before_any_launch(kw, msg):
    L = lib()
    a = dict(M=16, V=64, N=32, w=256, idx=512, dtype=2, bits=64)
    a.update(kw)
    rc = L.nn_embedding_fwd(a["w"], a["idx"], 1024, a["M"], a["V"], a["N"], 1.0, a["dtype"], a["bits"], None)
    assert rc != 0 and msg in L.nn_embedding_last_error().decode()
    with pytest.raises(RuntimeError, match=msg):
        check_embedding(rc)
    rc = L.nn_embedding_bwd(a["w"], a["idx"], 1024, 4096, 1 << 40, a["M"], a["V"], a["N"], 1.0, -1, a["dtype"], a["bits"], None)
    assert rc != 0 and msg in L.nn_embedding_last_error().decode()


def test_embedding_backward_workspace():
    L = lib()
    n = L.nn_embedding_bwd_workspace_size(8192, 50304, 768)
    # four sorted lists, the counts of 8 blocks, and two fp32 rows for each of 1024 chunks
    assert n == 4 * 4 * 8192 + 8 * 512 * 4 + 1024 * 2 * 768 * 4
    assert L.nn_embedding_bwd_workspace_size(0, 50304, 768) == 0 == L.nn_embedding_bwd_workspace_size(-1, 1, 1)
    assert L.nn_embedding_bwd(256, 512, 1024, 4096, n - 1, 8192, 50304, 768, 1.0, -1, 2, 64, None) != 0
    assert b"workspace too small" in L.nn_embedding_last_error()
    assert L.nn_embedding_bwd(256, 512, 1024, 4104, n, 8192, 50304, 768, 1.0, -1, 2, 64, None) != 0
    assert b"workspace must be 16-byte aligned" in L.nn_embedding_last_error()


def test_embedding_schema_and_fake():
    from nanonemo_amd.kernels.hip.embedding import embedding

    assert str(torch.ops.nanonemo.embedding.default._schema) == "nanonemo::embedding(Tensor idx, Tensor weight, float scale, SymInt padding_idx) -> Tensor"
    idx, w = torch.zeros(2, 5, dtype=torch.int64, device="meta"), torch.zeros(96, 64, dtype=torch.bfloat16, device="meta", requires_grad=True)
    out = embedding(idx, w, 8.0, -1)
    assert out.shape == (2, 5, 64) and out.dtype == torch.bfloat16 and out.is_contiguous()
    (dw,) = torch.autograd.grad(out, w, torch.empty_like(out))
    assert dw.shape == w.shape and dw.dtype == w.dtype


def test_embedding_refuses_what_it_cannot_run():
    from nanonemo_amd.kernels.hip.embedding import embedding

    idx, w = torch.zeros(3, dtype=torch.int64), torch.zeros(10, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        embedding(idx, w)
    for pad in (10, -11):
        with pytest.raises(ValueError, match="padding_idx"):
            embedding(idx, w, padding_idx=pad)


def test_capture_through_autograd_is_refused(monkeypatch):
    from nanonemo_amd.kernels.hip import embedding as emb

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    idx, w = torch.zeros(3, dtype=torch.int64), torch.zeros(10, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match="embedding: capturing"):
        emb.embedding(idx, w)
    with pytest.raises(RuntimeError, match="capturing"):
        emb._backward(None, w)
    with pytest.raises(RuntimeError, match="capturing"):
        emb._setup_context(None, (), w)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors"):  # nothing to record: on to the op's own checks
        emb.embedding(idx, w)


def test_model_options():
    with pytest.raises(ValueError, match="emb_kernel"):
        ModelConfig(emb_kernel="cuda")
    assert ModelConfig(emb_kernel="hip").any_hip and not ModelConfig(emb_scale=2.0).any_hip
    torch.manual_seed(0)
    plain, scaled = NanoNemo(ModelConfig(**SMALL)), NanoNemo(ModelConfig(**SMALL, emb_scale=8.0))
    assert type(plain.tok_emb) is torch.nn.Embedding
    scaled.load_state_dict(plain.state_dict())
    idx = torch.randint(0, 96, (2, 16))
    assert torch.equal(scaled.tok_emb(idx), plain.tok_emb(idx) * 8.0)
    assert not torch.equal(scaled(idx)[0], plain(idx)[0])
    # on the CPU the module is PyTorch's, whatever its kernel
    hip = NanoNemo(ModelConfig(**SMALL, emb_kernel="hip"))
    hip.load_state_dict(plain.state_dict())
    assert torch.equal(hip(idx)[0], plain(idx)[0])


# ---- distillation -------------------------------------------------------------------------------


@pytest.mark.parametrize(
    "kw, msg",
    [
        (dict(R=0), "invalid sizes"),
        (dict(R=1 << 22), "invalid sizes"),
        (dict(V=0), "invalid sizes"),
        (dict(V=393217), "invalid sizes"),
        (dict(T=0), "invalid sizes"),
        (dict(T=17), "invalid sizes"),
        (dict(sb=-1), "invalid strides"),
        (dict(st=1 << 40), "invalid strides"),
        (dict(k=0), "k must be in"),
        (dict(k=65), "k must be in"),
        (dict(V=1000, k=513), "k must be in"),
        (dict(tau=0.0), "temperature must be in"),
        (dict(tau=math.nan), "temperature must be in"),
        (dict(tau=2e4), "temperature must be in"),
        (dict(dtype=3), "dtype must be float16, bfloat16 or float32"),
        (dict(logits=257), "aligned to their type"),
        (dict(logits=None), "null pointer"),
        (dict(indices=None), "null pointer"),
    ],
)
def test_distill_c_abi_rejects_bad_arguments_before_any_launch(kw, msg):
    L = lib()
    a = dict(logits=256, T=16, sb=0, st=64, indices=1024, R=16, V=64, k=4, tau=1.0, dtype=1)
    a.update(kw)
    where = (a["logits"], a["T"], a["sb"], a["st"])
    size = (a["R"], a["V"], a["k"], a["tau"])
    rc = L.nn_top_logits(*where, 512, a["indices"], 2048, *size, a["dtype"], None)
    assert rc != 0 and msg in L.nn_distill_last_error().decode()
    with pytest.raises(RuntimeError, match=msg):
        check_distill(rc)
    rc = L.nn_distill_fwd(*where, 512, a["indices"], None, None, 2048, 4096, *size, 0.5, a["dtype"], 1, None)
    assert rc != 0 and msg in L.nn_distill_last_error().decode()
    rc = L.nn_distill_bwd(2048, *where, 512, a["indices"], None, 4096, 8192, *size, 0.5, a["dtype"], 1, None)
    assert rc != 0 and msg in L.nn_distill_last_error().decode()


def test_distill_c_abi_checks_of_the_loss():
    L = lib()
    assert L.nn_distill_stats_size(0) == 0 and L.nn_distill_stats_size(8192) == 8192 * 8 + 1
    for weight, value_dtype, out, msg in ((-0.1, 1, 8192, "weight must be in"), (math.nan, 1, 8192, "weight must be in"), (0.5, 3, 8192, "dtype must be"), (0.5, 1, 8193, "dlogits must be aligned")):
        rc = L.nn_distill_bwd(2048, 256, 16, 0, 64, 512, 1024, None, 4096, out, 16, 64, 4, 1.0, weight, 1, value_dtype, None)
        assert rc != 0 and msg in L.nn_distill_last_error().decode()


def test_distill_schemas_and_fakes():
    from nanonemo_amd.kernels.hip import distill as d

    assert str(torch.ops.nanonemo.top_logits.default._schema) == "nanonemo::top_logits(Tensor logits, SymInt k, float temperature) -> (Tensor, Tensor, Tensor)"
    assert str(torch.ops.nanonemo.distill_loss.default._schema) == (
        "nanonemo::distill_loss(Tensor logits, Tensor values, Tensor indices, Tensor? rest, Tensor? targets, float temperature, float weight) -> (Tensor, Tensor)")
    z = torch.empty(2, 5, 96, dtype=torch.bfloat16, device="meta", requires_grad=True)
    v, i, r = d.top_logits(z, 4, 2.0)
    assert v.shape == i.shape == (2, 5, 4) and r.shape == (2, 5) and (v.dtype, i.dtype, r.dtype) == (torch.bfloat16, torch.int64, torch.float32)
    assert not v.requires_grad
    loss = d.distill_loss(z, v, i, r, torch.empty(2, 5, dtype=torch.int64, device="meta"), 2.0, 0.5)
    assert loss.shape == () and loss.dtype == torch.float32
    (g,) = torch.autograd.grad(loss, z)
    assert g.shape == z.shape and g.dtype == z.dtype


def test_distill_refuses_what_it_cannot_run():
    from nanonemo_amd.kernels.hip import distill as d, host

    z, i = torch.zeros(3, 50), torch.zeros(3, 4, dtype=torch.int64)
    for call in (lambda: d.top_logits(z, 4), lambda: d.distill_loss(z, z[:, :4], i), lambda: host().distill_bwd(z[0, 0], z, z[:, :4], i, None, torch.zeros(22), 1.0, 1.0)):
        with pytest.raises(RuntimeError, match="CUDA tensors"):
            call()
    for call, msg in ((lambda: d.top_logits(z, 51), "k must be"), (lambda: d.top_logits(z, 4, -1.0), "temperature"), (lambda: d.distill_loss(z, z[:, :4], i, weight=0.5), "needs targets"),
                      (lambda: d.distill_loss(z, z[:, :4], i, weight=-1.0), "weight"), (lambda: d.distill_loss(z, z[:, :4].requires_grad_(), i), "no gradient"),
                      (lambda: d.distill_loss(z, z[:, :4], i, z[:, 0].requires_grad_()), "no gradient")):
        with pytest.raises(ValueError, match=msg):
            call()


def test_capture_of_the_loss_through_autograd_is_refused(monkeypatch):
    from nanonemo_amd.kernels.hip import distill as d

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    z, i = torch.zeros(3, 50, requires_grad=True), torch.zeros(3, 4, dtype=torch.int64)
    v = torch.zeros(3, 4)
    with pytest.raises(RuntimeError, match="distill_loss: capturing"):
        d.distill_loss(z, v, i)
    with pytest.raises(RuntimeError, match="capturing"):
        d._backward(None, z, None)
    with pytest.raises(RuntimeError, match="capturing"):
        d._setup_context(None, (), (z, z))
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors"):
        d.distill_loss(z, v, i)
    with pytest.raises(RuntimeError, match="CUDA tensors"):  # (takes no gradient)
        d.top_logits(z, 4)


def test_plain_distillation_of_a_model():
    torch.manual_seed(0)
    teacher, student = NanoNemo(ModelConfig(**SMALL)), NanoNemo(ModelConfig(**SMALL))
    idx = torch.randint(0, 96, (2, 16))
    y = idx.roll(-1, 1)
    y[:, 12:] = -100
    (batch,) = teacher_batches(teacher, [(idx, y)], 8, temperature=2.0, weight=0.25, amp_dtype=None)
    t = batch[2]
    full = teacher(idx)[0].detach()
    assert t.values.shape == t.indices.shape == (2, 16, 8) and t.rest.shape == (2, 16) and (t.temperature, t.weight) == (2.0, 0.25)
    logits, loss = student(*batch)
    # the definition, with the teacher's whole distribution: k = V and no rest
    p, q = torch.log_softmax(full / 2, -1), torch.log_softmax(logits / 2, -1)
    top, rest = torch.zeros(2, 16, 9), torch.zeros(2, 16, 9)
    inside = torch.zeros_like(p, dtype=torch.bool).scatter_(-1, t.indices, True)
    for o, lp in ((top, p), (rest, q)):
        o[..., :8], o[..., 8] = lp.gather(-1, t.indices), lp.masked_fill(inside, -math.inf).logsumexp(-1)
    kl = (top.exp() * (top - rest)).sum(-1)[y != -100].mean()
    torch.testing.assert_close(loss, 0.25 * 4 * kl + 0.75 * F.cross_entropy(logits.view(-1, 96), y.view(-1)))
    whole = Teacher(full, torch.arange(96).expand(2, 16, 96), None, 2.0, 1.0)
    torch.testing.assert_close(distill_loss(logits, whole, None), 4 * (p.exp() * (p - q)).sum(-1).mean())
    with pytest.raises(ValueError, match="needs targets"):
        student(idx, None, t)
    assert student(idx, None, t._replace(weight=1.0))[1].isfinite()
    loss, norm = train_step(student, make_optimizer(student), [batch], amp_dtype=None)
    assert loss.isfinite() and norm > 0


@pytest.mark.parametrize("kernel", ["torch", "hip"])
@pytest.mark.parametrize("how", ["script", "trace"])
def test_the_embedding_module_is_scripted_and_traced_as_pytorchs(kernel, how):
    from nanonemo_amd.model import Embedding

    m = Embedding(20, 8, 3.0, kernel, padding_idx=2)
    idx = torch.randint(0, 20, (3, 5))
    got = torch.jit.script(m) if how == "script" else torch.fx.symbolic_trace(m)
    ref = F.embedding(idx, m.weight, 2) * 3.0
    assert torch.equal(got(idx), ref) and torch.equal(m(idx), ref)
    (g,), (r,) = (torch.autograd.grad(f(idx).square().sum(), m.weight) for f in (got, lambda i: F.embedding(i, m.weight, 2) * 3.0))
    assert torch.equal(g, r) and not g[2].any()
