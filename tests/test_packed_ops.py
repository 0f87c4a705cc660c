"""CPU tests of the operators of packed sequences: the plan of the packed attention (what its kernels read and write by), the
boundary's checks, schemas and fake impls. No GPU compute is launched here."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

from nanonemo_amd.kernels.hip import host, lib

CASES = [
    ([], 4, 2), ([0], 4, 2), ([0, 0, 5, 0], 4, 1), ([1], 1, 1), ([63, 64, 65, 1, 127, 128, 129, 0], 12, 4), ([1024] * 8, 12, 4), ([1024] * 32, 12, 4),
    ([8192] + [37] * 60, 12, 4), ([5000, 1], 12, 1), ([4096, 300, 300], 8, 8), ([16] * 700, 12, 4), ([1, 2, 3] * 500, 4, 1), ([300] * 257, 12, 4),
    ([100000], 2, 1), ([8192, 8192], 12, 4),
]


def _c(lengths):
    return (ctypes.c_int64 * max(1, len(lengths)))(*lengths)


def _plan(lengths, H, KVH):
    words = lib().nn_fa_packed_plan_words(_c(lengths), len(lengths), H, KVH)
    plan = (ctypes.c_int32 * words)()
    assert lib().nn_fa_packed_plan(_c(lengths), len(lengths), H, KVH, plan, words) == 0
    return list(plan)


def _check_plan(lengths, H, KVH):
    """Every tile, unit, iteration and partial sum once, whole, and within its sequence and the workspace."""
    w, g, tokens = _plan(lengths, H, KVH), H // KVH, sum(lengths)
    magic, words, n, h, kvh, total, longest, ntiles, nunits, nsums, nslots, wpp, tiles, units, sums, positions, nshort, shorts = w[:18]
    assert (words, n, h, kvh, total, longest) == (len(w), len(lengths), H, KVH, tokens, max(lengths, default=0))
    assert tiles == 32 and units == tiles + 4 * ntiles and sums == units + 8 * nunits and shorts == sums + 8 * nsums
    assert positions == shorts + 4 * nshort and len(w) == positions + tokens and ntiles % 8 == 0 and wpp in (1, 4)
    assert w[positions:] == [t for n in lengths for t in range(n)]
    starts = [sum(lengths[:i]) for i in range(len(lengths))]

    few = [tuple(w[shorts + 4 * i : shorts + 4 * i + 4]) for i in range(nshort)]  # sequences of up to 64 tokens, or none of them
    upto = 64 if few or longest <= 64 else 0
    assert sorted(few) == sorted((s, n, t, 0) for s, n in zip(starts, lengths) if n <= upto for t in range(-(-n // 32)))
    starts, lengths = [s for s, n in zip(starts, lengths) if n > upto], [n for n in lengths if n > upto]

    got = [tuple(w[tiles + 4 * i : tiles + 4 * i + 4]) for i in range(ntiles)]
    real = [t for t in got if t[1]]
    assert got == real + [(0, 0, 0, 0)] * (ntiles - len(real))
    assert sorted(real) == sorted((s, n, b, j) for s, n in zip(starts, lengths) for b in range(-(-n // 128)) for j in range(KVH))
    assert [t[2] for t in real] == sorted((t[2] for t in real), reverse=True)  # the heaviest first

    entries = [tuple(w[units + 8 * i : units + 8 * i + 8]) for i in range(nunits)]
    joined = {(s, p, j): (ns, slot) for s, n, p, j, ns, _, slot, _ in (tuple(w[sums + 8 * i : sums + 8 * i + 8]) for i in range(nsums))}
    assert len(joined) == nsums
    seen, slots = {}, []
    for s, n, p, j, ns, sidx, slot, paired in entries:
        assert (s, n) in zip(starts, lengths) and n > 0 and 0 <= j < KVH and 0 <= sidx < ns <= 16
        nkb = -(-n // 64)
        mine = [p] + ([nkb - 1 - p] if paired and nkb - 1 - p > p else [])
        for u in mine:
            assert 0 <= u < nkb
            seen.setdefault((s, u, j), []).append((sidx, ns))
        if ns > 1:
            assert wpp == 4 and paired and slot == joined[s, p, j][1] + sidx and joined[s, p, j][0] == ns
            slots.append(slot)
            assert all(g * (nkb - u) // ns >= 0 for u in mine) and (ns + 1) * g * nkb < 2**31  # the kernel's 32-bit split bounds
    assert sorted(slots) == list(range(nslots)) and sum(ns for ns, _ in joined.values()) == nslots
    assert set(seen) == {(s, u, j) for s, n in zip(starts, lengths) for u in range(-(-n // 64)) for j in range(KVH)}
    for shares in seen.values():
        assert sorted(shares) == [(i, len(shares)) for i in range(len(shares))]
    rnd = lambda b: (b + 255) // 256 * 256  # noqa: E731
    plan = (ctypes.c_int32 * len(w))(*w)
    for D in (32, 64):
        assert lib().nn_fa_packed_bwd_workspace_size(plan, D) == 2 * rnd(4 * H * tokens) + nslots * 2 * 128 * D * 4
    return w[:18]


@pytest.mark.parametrize("lengths, H, KVH", CASES, ids=[f"{len(c[0])}x{max(c[0], default=0)}-{c[1]}-{c[2]}" for c in CASES])
def test_plan_covers_every_sequence_once(lengths, H, KVH):
    _check_plan(lengths, H, KVH)


@pytest.mark.parametrize("seed", range(12))
def test_plan_of_random_sequences(seed):
    rng = random.Random(seed)
    top = rng.choice([3, 70, 300, 2000, 9000])
    lengths = [int(top * rng.random() ** 3) for _ in range(rng.choice([1, 5, 60, 300]))]
    H, KVH = rng.choice([(12, 4), (4, 1), (8, 8), (16, 2), (1, 1)])
    _check_plan(lengths, H, KVH)


def test_plan_shares_out_the_work():
    # equal long sequences that fill the chip are not split; one long sequence is, also beside short ones, and short ones never
    assert _check_plan([1024] * 8, 12, 4)[10] == 0
    assert _check_plan([2048], 12, 4)[10] > 0
    assert _check_plan([4096] + [100] * 30, 12, 4)[10] > 0 and _check_plan([1000, 500], 12, 4)[10] == 0
    assert _check_plan([256], 12, 4)[8] == 16 and _check_plan([900, 1024], 12, 4)[8] == 124  # a block for each unit
    assert _check_plan([1024] * 32, 12, 4)[11] == 1  # a wave for each pair
    assert _check_plan([20, 64], 12, 4)[16] == 3 and _check_plan([20, 64, 65], 12, 4)[16] == 0  # short sequences alone,
    assert _check_plan([20] * 100 + [300], 12, 4)[16] == 100  # or many of them


@pytest.mark.parametrize(
    "lengths, H, KVH, msg",
    [([3, -1], 4, 2, "sequence 1 has the length -1"), ([3], 4, 3, "group evenly"), ([3], 0, 1, "invalid sizes"), ([3], 4, 0, "invalid sizes"),
     ([1 << 30], 1, 1, "sizes too large"), ([1 << 29, 1 << 29], 1, 1, "sizes too large"), ([1 << 29], 64, 1, "sizes too large")],
)
def test_plan_refuses(lengths, H, KVH, msg):
    assert lib().nn_fa_packed_plan_words(_c(lengths), len(lengths), H, KVH) == 0
    assert msg in lib().nn_fa_last_error().decode()
    with pytest.raises(RuntimeError, match=msg):
        host().packed_plan(lengths, H, KVH)


def test_c_abi_rejects_bad_arguments_before_any_launch():
    L = lib()
    lengths = [5, 9]
    words = L.nn_fa_packed_plan_words(_c(lengths), 2, 4, 2)
    plan = (ctypes.c_int32 * words)()
    assert L.nn_fa_packed_plan(_c(lengths), 2, 4, 2, plan, words - 1) != 0 and b"words" in L.nn_fa_last_error()
    assert L.nn_fa_packed_plan(_c(lengths), 2, 4, 2, None, words) != 0
    assert L.nn_fa_packed_plan_words(None, 2, 4, 2) == 0 and L.nn_fa_packed_plan_words(_c(lengths), -1, 4, 2) == 0
    assert L.nn_fa_packed_fwd(16, 16, 16, 16, 16, None, plan, 16, 64, None, 1, 0.125, None) != 0 and b"not a plan" in L.nn_fa_last_error()
    assert L.nn_fa_packed_plan(_c(lengths), 2, 4, 2, plan, words) == 0

    def fwd(q=16, o=16, lse=16, rest=None, p=plan, dp=16, D=64, strides=None, dt=1):
        s = None if strides is None else (ctypes.c_int64 * 6)(*strides)
        return L.nn_fa_packed_fwd(q, 16, 16, o, lse, rest, p, dp, D, s, dt, 0.125, None), L.nn_fa_last_error().decode()

    for kw, msg in ((dict(q=None), "null"), (dict(o=None), "null"), (dict(q=8), "16-byte"), (dict(rest=4), "16-byte"), (dict(p=None), "null plan"), (dict(dp=None), "null plan"), (dict(dp=20), "16-byte"),
                    (dict(D=48), "head_dim"), (dict(dt=2), "float16 or bfloat16"), (dict(strides=[64, 256, 64, 100, 64, 256]), "multiples of 8"),
                    (dict(strides=[64, 32, 64, 128, 64, 256]), "smaller than head_dim"), (dict(strides=[64, 1 << 28, 64, 128, 64, 256]), "too large")):
        rc, got = fwd(**kw)
        assert rc != 0 and msg in got, (kw, got)

    def bwd(ws=256, n=1 << 20, scale=0.125, q=16, rest=None):
        return L.nn_fa_packed_bwd(16, q, 16, 16, 16, 16, rest, 16, 16, 16, ws, n, plan, 16, 64, None, 1, scale, None), L.nn_fa_last_error().decode()

    for kw, msg in ((dict(ws=None), "null workspace"), (dict(ws=128), "256-byte"), (dict(n=8), "too small"), (dict(scale=0.0), "positive"), (dict(q=None), "null"), (dict(q=8), "16-byte"), (dict(rest=8), "16-byte")):
        rc, got = bwd(**kw)
        assert rc != 0 and msg in got, (kw, got)
    words = L.nn_fa_packed_plan_words(_c([0, 0]), 2, 4, 2)  # nothing to do
    empty = (ctypes.c_int32 * words)()
    assert L.nn_fa_packed_plan(_c([0, 0]), 2, 4, 2, empty, words) == 0
    assert L.nn_fa_packed_fwd(None, None, None, None, None, None, empty, 16, 64, None, 1, 0.125, None) == 0
    assert L.nn_fa_packed_bwd_workspace_size(empty, 64) == 0


def _norm_args(**kw):
    a = dict(q=16, k=16, wq=16, wk=16, cos=16, sin=16, rows=8, pos=None, bits=64, period=4, yq=16, yk=16, M=4, H=4, KVH=2, D=64, s=[256, 64, 128, 64, 256, 64, 128, 64], eps=1e-5, dt=1)
    a.update(kw)
    a["s"] = None if a["s"] is None else (ctypes.c_int64 * 12)(*a["s"])
    return a


@pytest.mark.parametrize(
    "kw, msg",
    [(dict(D=24), "multiple of 16"), (dict(D=272), "up to 256"), (dict(dt=3), "float16, bfloat16 or float32"), (dict(H=0), "invalid sizes"), (dict(KVH=0), "invalid sizes"), (dict(M=-1), "invalid sizes"),
     (dict(rows=3), "exceeds the 3 rows"), (dict(rows=0), "no rows"), (dict(s=None), "null strides"), (dict(s=[256, 60, 128, 64, 256, 64, 128, 64]), "multiples of 8"), (dict(wq=None), "null"), (dict(cos=8), "16-byte"),
     (dict(q=8), "16-byte"), (dict(yk=None), "null"), (dict(period=0), "period"), (dict(pos=16, bits=16), "int32 or int64"), (dict(pos=12, bits=64), "aligned"), (dict(M=1 << 31, rows=1 << 32, period=1 << 30), "too large"),
     (dict(M=1 << 27, rows=1 << 32, period=1 << 30), "too large")],
)
def test_qk_norm_c_abi_rejects_bad_arguments_before_any_launch(kw, msg):
    a, L = _norm_args(**kw), lib()
    rc = L.nn_qk_norm_rope_fwd(a["q"], a["k"], a["wq"], a["wk"], a["cos"], a["sin"], a["rows"], a["pos"], a["bits"], a["period"], a["yq"], a["yk"], a["M"], a["H"], a["KVH"], a["D"], a["s"], a["eps"], a["dt"], None)
    assert rc != 0 and msg in L.nn_qk_norm_last_error().decode()
    s = None if a["s"] is None else (ctypes.c_int64 * 12)(*([64] * 8 + list(a["s"])[:4] if "s" not in kw else list(a["s"])))
    rc = L.nn_qk_norm_rope_bwd(16, 16, a["q"], a["k"], a["wq"], a["wk"], a["cos"], a["sin"], a["rows"], a["pos"], a["bits"], a["period"], a["yq"], a["yk"], 16, 16, 256, 1 << 30, a["M"], a["H"], a["KVH"], a["D"], s, a["eps"],
                               a["dt"], None)
    assert rc != 0 and msg in L.nn_qk_norm_last_error().decode()


def test_qk_norm_workspace():
    L = lib()
    assert L.nn_qk_norm_rope_bwd_workspace_size(0, 4, 2, 64) == 0
    assert L.nn_qk_norm_rope_bwd_workspace_size(-1, 4, 2, 64) == 0
    for M, H, KVH, D in ((1, 1, 1, 16), (5, 12, 4, 64), (8192, 12, 4, 64), (131072, 9, 3, 128), (1 << 20, 64, 1, 256)):
        n = L.nn_qk_norm_rope_bwd_workspace_size(M, H, KVH, D)
        assert n % (4 * D) == 0 and 2 * 4 * D <= n <= 4096 * 4 * D  # at least a block for queries and one for keys
    a = _norm_args()
    rc = L.nn_qk_norm_rope_bwd(16, 16, 16, 16, 16, 16, 16, 16, 8, None, 0, 4, 16, 16, 16, 16, 256, 8, 4, 4, 2, 64, (ctypes.c_int64 * 12)(*[64] * 12), 1e-5, 1, None)
    assert rc != 0 and b"workspace" in L.nn_qk_norm_last_error() and a


def _packing(lengths, H, KVH):
    from nanonemo_amd.kernels.hip.packed import Packing

    return Packing(lengths, H, KVH, device="cpu")


def test_packing():
    p = _packing([3, 0, 5], 4, 2)
    assert (p.lengths, p.tokens, p.longest, p.heads, p.kv_heads, p.device.type) == ((3, 0, 5), 8, 5, 4, 2, "cpu")
    assert p.positions.tolist() == [0, 1, 2, 0, 1, 2, 3, 4] and p.positions.dtype == torch.int32
    assert _packing(torch.tensor([2, 2]), 4, 2).positions.tolist() == [0, 1, 0, 1] and _packing([], 4, 2).tokens == 0
    for lengths in ([3, -2], [3.5], ["x"], torch.tensor([1.0])):
        with pytest.raises((RuntimeError, TypeError)):
            _packing(lengths, 4, 2)


def test_schemas_and_fakes():
    from nanonemo_amd.kernels.hip.packed import flash_attn_packed
    from nanonemo_amd.kernels.hip.qk_norm import qk_norm_rope

    ops = torch.ops.nanonemo
    assert str(ops.flash_attn_packed.default._schema) == "nanonemo::flash_attn_packed(Tensor q, Tensor k, Tensor v, Tensor plan, Tensor plan_host, bool backward) -> (Tensor, Tensor, Tensor)"
    assert str(ops.qk_norm_rope.default._schema) == (
        "nanonemo::qk_norm_rope(Tensor q, Tensor k, Tensor q_weight, Tensor k_weight, Tensor cos, Tensor sin, Tensor? positions, float eps) -> (Tensor, Tensor)")

    def meta(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device="meta", requires_grad=True)

    q, k, v = meta(8, 4, 64), meta(8, 2, 64), meta(8, 2, 64)
    wq, wk = meta(64, dtype=torch.float32), meta(64, dtype=torch.float32)
    table = torch.zeros(16, 32, device="meta")
    rq, rk = qk_norm_rope(q.transpose(0, 1).contiguous().transpose(0, 1), k, wq, wk, table, table)
    o = flash_attn_packed(rq, rk, v, _packing([3, 5], 4, 2))
    assert o.shape == q.shape and o.dtype == q.dtype and o.is_contiguous() and rq.is_contiguous()
    for t, g in zip((q, k, v, wq, wk), torch.autograd.grad(o, (q, k, v, wq, wk), torch.empty_like(o))):
        assert g.shape == t.shape and g.dtype == t.dtype


def test_refuse_what_they_cannot_run():
    from nanonemo_amd.kernels.hip.packed import flash_attn_packed
    from nanonemo_amd.kernels.hip.qk_norm import qk_norm_rope

    q, k, t, w = torch.zeros(8, 4, 64), torch.zeros(8, 2, 64), torch.zeros(8, 32), torch.ones(64)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        flash_attn_packed(q.half(), k.half(), k.half(), _packing([3, 5], 4, 2))
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        qk_norm_rope(q, k, w, w, t, t)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            flash_attn_packed(dual, k, k, _packing([3, 5], 4, 2))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            qk_norm_rope(dual, k, w, w, t, t)


def test_capture_through_autograd_is_refused(monkeypatch):
    from nanonemo_amd.kernels.hip import packed, qk_norm

    packing = _packing([3, 5], 4, 2)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    q, k, t, w = torch.zeros(8, 4, 64, requires_grad=True), torch.zeros(8, 2, 64), torch.zeros(8, 32), torch.ones(64, requires_grad=True)
    with pytest.raises(RuntimeError, match="flash_attn_packed: capturing"):
        packed.flash_attn_packed(q, k, k, packing)
    with pytest.raises(RuntimeError, match="qk_norm_rope: capturing"):
        qk_norm.qk_norm_rope(q.detach(), k, w, w, t, t)
    for m in (packed, qk_norm):
        with pytest.raises(RuntimeError, match="capturing"):
            m._backward(None, q, None)
        with pytest.raises(RuntimeError, match="capturing"):
            m._setup_context(None, (), q)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensors"):  # nothing to record: on to the op's own checks
        packed.flash_attn_packed(q, k, k, packing)
    with pytest.raises(RuntimeError, match="while a HIP graph is captured"):
        packed.Packing([3], 4, 2, device="cuda")


SMALL = dict(n_layers=2, d_model=128, n_heads=4, n_kv_heads=2, d_ff=256, vocab_size=97, max_seq_len=64)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_a_packed_model_is_the_model_on_each_sequence(qk_norm):
    from nanonemo_amd.model import ModelConfig, NanoNemo

    torch.manual_seed(0)
    model = NanoNemo(ModelConfig(**SMALL, qk_norm=qk_norm))
    assert ("blocks.0.attn.q_norm.weight" in model.state_dict()) == qk_norm
    if qk_norm:
        for p in (model.blocks[0].attn.q_norm.weight, model.blocks[1].attn.k_norm.weight):
            torch.nn.init.normal_(p, 1.0, 0.2)
    lengths = [5, 0, 1, 64, 20]
    idx, y = (torch.randint(0, 97, (2, 45)) for _ in range(2))
    y[0, 4] = -100
    packing = model.pack(lengths)
    logits, loss = model(idx, y, None, packing)
    alone = torch.cat([model(t[None])[0][0] for t in idx.flatten().split(lengths) if len(t)])
    # the same fp32 sums in another order: 2^-24 of about 1 each, some hundred of them
    torch.testing.assert_close(logits.view(90, -1), alone, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(loss, torch.nn.functional.cross_entropy(alone, y.flatten()), rtol=1e-5, atol=1e-5)
    assert model(idx, None, None, packing)[1] is None
    t = model.teach(idx, 3, packing=packing)
    assert torch.equal(t.indices, logits.topk(3).indices)
    loss = model(idx, y, t, packing)[1]
    loss.backward()
    assert all(p.grad is not None for p in model.parameters())
    with pytest.raises(ValueError, match="90 tokens, but a packing of 89"):
        model(idx, None, None, model.pack([64, 25]))
    with pytest.raises(ValueError, match="max_seq_len"):
        model(idx, None, None, model.pack([65, 25]))


def test_a_packing_without_tokens_is_refused_by_the_model():
    from nanonemo_amd.model import ModelConfig, NanoNemo

    model = NanoNemo(ModelConfig(n_layers=1, d_model=64, n_heads=2, n_kv_heads=1, d_ff=64, vocab_size=64, max_seq_len=32))
    for lengths in ([], [0, 0]):
        with pytest.raises(ValueError, match="without tokens"):
            model(torch.zeros(1, 0, dtype=torch.long), None, None, model.pack(lengths))


@pytest.mark.parametrize("qk_norm", [False, True])
def test_a_packed_attention_layer_takes_one_row_and_its_tokens_tables(qk_norm):
    """Two rows would take the tables' first rows each, whole tables those of a single sequence."""
    from nanonemo_amd.model import Attention, ModelConfig, rope_tables

    torch.manual_seed(0)
    m = Attention(ModelConfig(**SMALL, qk_norm=qk_norm))
    lengths = [13, 7]
    packing, x = _packing(lengths, 4, 2), torch.randn(1, 20, 128)
    tables = rope_tables(32, 64, 10000.0)
    cos, sin = (t[packing.positions] for t in tables)
    alone = torch.cat([m(t, *tables) for t in x.split(lengths, 1)], 1)
    torch.testing.assert_close(m(x, cos, sin, packing), alone, rtol=1e-4, atol=1e-5)
    for bad in ((x.view(2, 10, 128), cos, sin), (x, *tables), (x, cos, tables[1]), (x, cos[:19], sin[:19])):
        with pytest.raises(ValueError, match="one row, with a row of cos and sin for each"):
            m(*bad, packing)


def test_a_plan_cut_short_is_refused():
    from nanonemo_amd.kernels.hip import host
    from nanonemo_amd.kernels.hip.packed import Packing

    plan = Packing([5, 9], 2, 1, device="cpu").plan_host
    q, k = torch.zeros(14, 2, 64, dtype=torch.bfloat16), torch.zeros(14, 1, 64, dtype=torch.bfloat16)
    for n in (0, 16, 31, 32, len(plan) - 1):
        with pytest.raises(RuntimeError, match="must be a Packing's"):
            host().packed_fwd(q, k, k, plan[:n], plan[:n], False)


def test_packed_batches():
    from nanonemo_amd.model import ModelConfig, NanoNemo
    from nanonemo_amd.train import packed_batches, synthetic_documents, teacher_batches, train_step

    model = NanoNemo(ModelConfig(**SMALL))
    docs = [torch.arange(n) % 97 for n in (10, 1, 0, 2, 150, 33)]
    batches = packed_batches(model, docs, 80)
    assert [p.lengths for *_, p in batches] == [(9, 1, 64), (64,), (21, 32)]
    for x, y, none, p in batches:
        assert none is None and x.shape == y.shape == (1, p.tokens) and torch.equal(y, (x + 1) % 97)
    assert torch.equal(batches[1][0][0], torch.arange(64, 128) % 97)  # a long document goes on where it was cut
    assert packed_batches(model, [], 80) == []
    assert [p.lengths for *_, p in packed_batches(model, docs[:1], 4)] == [(4,), (4,), (1,)]
    docs = synthetic_documents(3, 80, 20, 97)
    assert sum(len(d) - 1 for d in docs) >= 240 and max(int(d.max()) for d in docs) < 97
    student = NanoNemo(ModelConfig(**SMALL))
    opt = torch.optim.SGD(student.parameters(), 0.1)
    for some in (batches[:2], teacher_batches(model, batches[:2], 3, amp_dtype=None)):
        loss, norm = train_step(student, opt, some, amp_dtype=None)
        assert loss.isfinite() and norm > 0


def test_a_micro_batch_that_has_a_teacher_gets_no_other():
    from nanonemo_amd.model import ModelConfig, NanoNemo
    from nanonemo_amd.train import packed_batches, synthetic_documents, teacher_batches

    model = NanoNemo(ModelConfig(**SMALL))
    packed = packed_batches(model, synthetic_documents(1, 80, 20, 97), 80)
    x, y = (torch.randint(0, 97, (2, 16)) for _ in range(2))
    for batches in ([(x, y)], [(x, y, None)], packed):
        taught = teacher_batches(model, batches, 3, amp_dtype=None)
        assert all(t[2].indices.shape == (*t[0].shape, 3) and t[3:] == b[3:] for t, b in zip(taught, batches))
        with pytest.raises(ValueError, match="has a teacher already"):
            teacher_batches(model, taught, 3, amp_dtype=None)


@pytest.mark.parametrize("hd", [256, 272])
def test_heads_past_the_norm_kernel_s_size_are_normalised_by_their_modules(hd):
    """The rotation's kernel takes larger heads than the norm's with the rotation, whose calls they would make an error."""
    from nanonemo_amd.model import Attention, ModelConfig, rope, rope_tables

    torch.manual_seed(0)
    sizes = dict(d_model=2 * hd, n_heads=2, n_kv_heads=1, d_ff=32, vocab_size=32, max_seq_len=9, qk_norm=True)
    plain, m = Attention(ModelConfig(**sizes)), Attention(ModelConfig(**sizes, rope_kernel="hip"))
    m.load_state_dict(plain.state_dict())
    with_norm = []
    m._rope_qk = lambda q, k, cos, sin: (rope(q, cos, sin, 1), rope(k, cos, sin, 1))  # (there is no GPU here)
    m._qk_norm_rope = lambda q, k, wq, wk, cos, sin, eps: with_norm.append(hd) or m._rope_qk(m.q_norm(q), m.k_norm(k), cos, sin)
    x, tables = torch.randn(2, 9, 2 * hd), rope_tables(hd, 9, 10000.0)
    torch.testing.assert_close(m(x, *tables), plain(x, *tables), rtol=1e-5, atol=1e-6)
    assert bool(with_norm) == (hd <= 256)


@pytest.mark.parametrize("seed", range(20))
def test_shares_of_split_pairs(seed):
    """A pair's blocks keep 8 iterations (query head, query tile) each at least, and their shares of each of its units, in the
    kernel's arithmetic, are the unit's iterations once. Pairs alone are split, and where that takes 64 iterations off a block."""
    rng = random.Random(seed)
    H, KVH = rng.choice([(12, 4), (4, 1), (8, 8), (16, 2), (1, 1), (12, 1)])
    lengths = [rng.choice([2048, 4096, 8192, 20000])] + [rng.randint(1, rng.choice([100, 600, 2000])) for _ in range(rng.choice([0, 3, 30]))]
    w, g = _plan(lengths, H, KVH), H // KVH
    upto = 64 if w[16] else 0
    # (query head, query tile) iterations of all units of 64 keys over 256 CUs
    even = sum(g * nkb * (nkb + 1) // 2 * KVH for nkb in (-(-n // 64) for n in lengths if n > upto)) // 256
    split = 0
    for i in range(w[8]):
        _, n, pj, _, ns, sidx, _, paired = w[w[13] + 8 * i : w[13] + 8 * i + 8]
        nkb = -(-n // 64)
        both = paired and nkb - 1 - pj > pj
        units = [g * (nkb - pj)] + ([g * (pj + 1)] if both else [])
        assert paired or ns == 1
        if ns > 1:
            split += sidx == 0
            assert sum(units) // ns >= 8 and sum(units) - even >= 64
        if sidx == 0:
            for it in units:
                shares = [(s * it // ns, (s + 1) * it // ns) for s in range(ns)]
                assert shares[0][0] == 0 and shares[-1][1] == it and all(a[1] == b[0] and a[0] <= a[1] for a, b in zip(shares, shares[1:]))
                assert (ns + 1) * it < 2**31
    assert split == w[9]
