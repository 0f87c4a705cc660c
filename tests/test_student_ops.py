"""CPU tests of the operators at the ends of a training step (embedding): schemas, fake impls, argument checks at the C ABI
and in the public functions, and the model's options. No GPU compute is launched here."""

from __future__ import annotations

import pytest
import torch

from nanonemo_amd.kernels.hip import check_embedding, lib
from nanonemo_amd.model import ModelConfig, NanoNemo

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
