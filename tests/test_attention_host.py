"""Host side of packed attention and the residual norm, without a GPU: lengths,
tiles, buckets and the refusals that come before any launch."""

from __future__ import annotations

import math

import pytest
import torch

import kanforge_b200 as kb
from kanforge_b200.attention import relative_buckets


def test_sequences_tables_and_refusals():
    s = kb.PackedSequences([3, 0, 5], [4, 2, 5], device="cpu")
    assert s.table.tolist() == [[0, 3, 0, 4], [3, 0, 4, 2], [3, 5, 6, 5]]
    assert (s.total_q, s.total_kv, len(s)) == (8, 11, 3)
    with pytest.raises(ValueError):
        kb.PackedSequences([1, -1], device="cpu")
    with pytest.raises(ValueError):
        kb.PackedSequences([1], [1, 2], device="cpu")
    with pytest.raises(ValueError):
        kb.PackedSequences([1 << 30, 1 << 30], device="cpu")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows", [1, 16, 64])
def test_tiles_cover_every_row_once_with_the_most_work_first(rows, causal):
    q_lens, kv_lens = [0, 1, 64, 65, 200], [3, 9, 64, 30, 300]
    s = kb.PackedSequences(q_lens, kv_lens, device="cpu")
    for side, lens in (("q", q_lens), ("k", kv_lens)):
        tiles = [tuple(t) for t in s.tiles(side, rows, causal).tolist()]
        assert sorted(tiles) == [(i, t) for i, n in enumerate(lens) for t in range(-(-n // rows))]
        cost = []
        for i, t in tiles:
            off = kv_lens[i] - q_lens[i]
            if side == "q":
                cost.append(max(0, min(kv_lens[i], (t + 1) * rows + off)) if causal else kv_lens[i])
            else:
                cost.append(max(0, q_lens[i] - max(0, t * rows - off)) if causal else q_lens[i])
        assert cost == sorted(cost, reverse=True)


@pytest.mark.parametrize("n,span,both", [(32, 128, True), (32, 128, False), (8, 20, True), (4, 3, True), (2, 2, False),
                                         (64, 2048, False)])
def test_buckets_follow_the_logarithm(n, span, both):
    got = relative_buckets(n, span, both)
    assert len(got) == 2 * span + 1 and min(got) == 0 and max(got) == n - 1
    one = n // 2 if both else n
    exact = one // 2
    for d in range(-span, span + 1):
        dist = abs(d) if both else max(0, d)
        if dist < exact:
            want = dist
        else:
            # 1e-9: the exact floor where the logarithm is a whole number
            want = min(one - 1, exact + int(math.log(dist / exact) / math.log(span / exact) * (one - exact) + 1e-9))
        assert got[d + span] == want + (one if both and d < 0 else 0), d


def test_bias_module_looks_up_and_refuses():
    b = kb.RelativeBias(3, 8, 16, bidirectional=False)
    with torch.no_grad():
        b.weight.copy_(torch.arange(24.0).reshape(8, 3))
    assert b(torch.tensor([0, 1, 500, -4])).tolist() == [[0, 1, 2], [3, 4, 5], [21, 22, 23], [0, 1, 2]]
    assert set(b.state_dict()) == {"weight"}
    for args in ((3, 1), (3, 7), (3, 300), (3, 32, 8), (3, 32, 4096), (0, 32)):
        with pytest.raises(ValueError):
            kb.RelativeBias(*args)


def test_cpu_tensors_raise():
    t = torch.randn(4, 2, 16)
    with pytest.raises(RuntimeError):
        kb.attention(t, t, t, kb.PackedSequences([4], device="cpu"))
    with pytest.raises(RuntimeError):
        kb.attention_decode(t, t[None], t[None], torch.ones(4, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        kb.residual_norm(t, t, torch.ones(16))


def test_entry_points_check_their_arguments_before_any_cuda_call():
    import ctypes

    from kanforge_b200 import _lib

    lib = _lib.load()
    d = _lib.AttentionDesc(heads=4, kv_heads=3, dim=64)
    assert lib.kf_attention_fwd(*[None] * 4, 1, *[None] * 5, ctypes.byref(d), None) == 1
    assert "do not divide" in _lib.last_error()
    d = _lib.AttentionDesc(heads=4, kv_heads=2, dim=65)
    assert lib.kf_attention_fwd(*[None] * 4, 1, *[None] * 5, ctypes.byref(d), None) == 1
    d = _lib.DecodeDesc(heads=4, kv_heads=2, dim=64, batch=1, capacity=8)
    assert lib.kf_attention_decode(*[None] * 7, ctypes.byref(d), None) == 1
    d = _lib.ResidualNormDesc(width=9000)
    x = ctypes.c_void_p(16)
    assert lib.kf_residual_norm_fwd(x, *[None] * 2, x, *[None] * 6, 1, ctypes.byref(d), None) == 1
    assert "outside" in _lib.last_error()


def test_transformer_refusals_and_cache():
    for bad in (dict(dim=48, depth=0, heads=6), dict(dim=48, depth=1, heads=5), dict(dim=48, depth=1, heads=12),
                dict(dim=272, depth=1, heads=2), dict(dim=48, depth=1, heads=6, kv_heads=4)):
        with pytest.raises(ValueError):
            kb.KANTransformer(**bad)
    m = kb.KANTransformer(48, 2, 6, 2, 64)
    assert m.bias.heads == 6 and not m.bias.bidirectional
    assert kb.KANTransformer(48, 1, 6, num_buckets=0).bias is None
    cache = m.new_cache(3, 4)
    assert cache.k.shape == cache.v.shape == (2, 3, 4, 2, 8)
    seq, slot = cache.begin([2, 0, 3])
    assert seq.tolist() == [0, 0, 2, 2, 2] and slot.tolist() == [0, 1, 0, 1, 2]
    seq, slot = cache.step()
    assert seq.tolist() == [0, 1, 2] and slot.tolist() == [2, 0, 3] and cache.lengths.tolist() == [3, 1, 4]
    with pytest.raises(ValueError):
        cache.step()
    for lens in ([1, 2], [1, 2, 5], [1, -1, 2]):
        with pytest.raises(ValueError):
            cache.begin(lens)
    with pytest.raises(ValueError):
        kb.KVCache(1, 0, 4, 2, 8)
    both = kb.KANTransformer(48, 1, 6, causal=False)
    with pytest.raises(ValueError):
        both.decode(torch.zeros(3, 48), both.new_cache(3, 4))


def test_backward_reads_saved_tensors_by_the_strides_they_have(monkeypatch):
    """Saved tensors may come back in another layout (offloaded to the host, say): here views of one
    projection come back contiguous."""
    import sys

    module = sys.modules["kanforge_b200.attention"]  # the package's name of it is the function
    calls = []
    monkeypatch.setattr(module, "_raw_stream", lambda t: 0)
    monkeypatch.setattr(module, "_launch", lambda name, *args, **kw: calls.append((name, args[-2]._obj)))
    seqs = kb.PackedSequences([3, 2], device="cpu")
    for contiguous, rows in ((False, (128, 128, 128)), (True, (64, 32, 32))):
        qkv = torch.randn(5, 8, 16).bfloat16().requires_grad_()
        pack = (lambda t: t.clone(memory_format=torch.contiguous_format)) if contiguous else (lambda t: t)
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            out = module._Attention.apply(*qkv.split([4, 2, 2], 1), None, seqs, True, 0.25, None)
        torch.autograd.grad(out, qkv, torch.ones_like(out))
        (fwd, f), (bwd, b) = calls
        calls.clear()
        assert (fwd, bwd) == ("kf_attention_fwd", "kf_attention_bwd")
        assert (f.q_row, f.k_row, f.v_row) == (128, 128, 128) and (b.q_row, b.k_row, b.v_row) == rows


def test_steps_the_host_does_not_count_stay_in_the_cache():
    """A step replayed from a CUDA graph advances the lengths on the device alone."""
    cache = kb.KVCache(1, 3, 4, 2, 8)
    cache.begin([2, 0, 4])
    for n in range(1, 6):
        cache.longest = 0  # what the host knows of replays
        seq, slot = cache.step()
        assert seq.tolist() == [0, 1, 2] and slot.tolist() == [min(2 + n - 1, 3), min(n - 1, 3), 3]
        assert cache.lengths.tolist() == [2 + n, n, 4 + n]  # above the capacity: a token too many


def test_refused_prompts_and_tokens_leave_the_cache_as_it_was():
    m = kb.KANTransformer(48, 2, 6, 2, 64)
    cache = m.new_cache(3, 8)
    cache.begin([2, 1, 3])
    cache.k.zero_(), cache.v.zero_()
    others = (kb.KVCache(1, 3, 8, 2, 8), kb.KVCache(2, 3, 8, 6, 8), kb.KVCache(2, 3, 8, 2, 16), kb.KVCache(2, 3, 8, 2, 8, device="meta"))
    for c in (cache, *others):
        bad = 1 if c is cache else 3
        with pytest.raises(ValueError):
            m.decode(torch.randn(bad, 48), c)  # one row would be stored for all three sequences
        with pytest.raises(ValueError):
            m.prefill(torch.randn(1 if c is cache else 5, 48), [2, 1, 2], c)
        assert c.longest == (3 if c is cache else 0)
    assert cache.lengths.tolist() == [2, 1, 3] and not cache.k.any() and not cache.v.any()


def test_bias_buckets_survive_every_way_a_module_moves():
    want = relative_buckets(8, 16, True)

    def right(b):
        return b.buckets.dtype == torch.int32 and b.buckets.device == b.weight.device and b.buckets.tolist() == want

    b = kb.RelativeBias(3, 8, 16, device="meta").to_empty(device="cpu")
    assert right(b)
    with torch.device("meta"):
        m = kb.KANTransformer(48, 1, 6, causal=False, num_buckets=8, max_distance=16)
    assert right(m.to_empty(device="cpu").bias)
    b.buckets.fill_(1 << 30)
    assert right(b.to_empty(device="cpu")) and right(b.type(torch.float64)) and right(b.bfloat16())
    kept = b.buckets
    assert b.to("cpu").buckets is kept  # a move that moves nothing: what a CUDA graph holds stays
    # weights of a checkpoint assigned to a model without memory
    b = kb.RelativeBias(3, 8, 16, device="meta")
    b.load_state_dict({"weight": torch.randn(8, 3)}, assign=True)
    assert b(torch.tensor([0, -20])).shape == (2, 3) and right(b)


def test_bias_whose_weight_has_another_shape_is_refused():
    from kanforge_b200.attention import _check_bias

    b = kb.RelativeBias(3, 8, 16)
    _check_bias(b, 3, torch.device("cpu"))
    b.weight = torch.nn.Parameter(torch.zeros(4, 3))
    with pytest.raises(ValueError):
        _check_bias(b, 3, torch.device("cpu"))
    b.weight = torch.nn.Parameter(torch.zeros(8, 3))
    b.buckets = b.buckets[:5]
    _check_bias(b, 3, torch.device("cpu"))
    assert b.buckets.tolist() == relative_buckets(8, 16, True)
    with pytest.raises(ValueError):
        _check_bias(b, 2, torch.device("cpu"))
    with pytest.raises(TypeError):
        _check_bias(b.half(), 3, torch.device("cpu"))


def test_entry_points_refuse_pointers_that_would_fault():
    import ctypes

    from kanforge_b200 import _lib

    lib, p, odd = _lib.load(), ctypes.c_void_p(64), ctypes.c_void_p(68)
    # the statistics are read and written 16 bytes at a time
    d = ctypes.byref(_lib.ResidualNormDesc(width=8, residual_scale=1.0))
    assert lib.kf_residual_norm_fwd(p, None, None, p, None, None, None, None, p, odd, 1, d, None) == 1
    assert "16 bytes" in _lib.last_error()
    assert lib.kf_residual_norm_bwd(p, None, None, p, None, None, odd, p, p, p, *[None] * 6, p, 1, d, None) == 1
    assert "16 bytes" in _lib.last_error()
    # both passes read the rows of both sides, whichever tiles are given
    for dtype, rest in ((0, None), (1, p)):
        d = ctypes.byref(_lib.AttentionDesc(tq=4, tk=4, q_row=64, q_head=64, k_row=64, k_head=64, v_row=64, v_head=64, heads=1,
                                            kv_heads=1, dim=64, dtype=dtype, scale=1.0))
        for missing in range(7):  # q, k, v, o, dout, lse, workspace
            q, k, v, o, g, lse, ws = (None if i == missing else p for i in range(7))
            for n_q, n_k in ((0, 1), (1, 0), (1, 1)):
                assert lib.kf_attention_bwd(q, k, v, o, rest, g, lse, p, n_q, p, n_k, None, None, p, p, p, None, ws, d, None) == 1, missing
                assert "null argument" in _lib.last_error()


def test_sequences_copy_and_pickle_after_use():
    """What is kept for calls stays behind: addresses, and descriptors that do not copy."""
    import copy
    import pickle

    from kanforge_b200.attention import _plan

    seqs = kb.PackedSequences([3, 2], [4, 2], device="cpu")
    q, k = torch.randn(5, 4, 16), torch.randn(6, 2, 16)
    _plan(seqs, q, k, k, True, 0.25, None)
    for other in (copy.copy(seqs), copy.deepcopy(seqs), pickle.loads(pickle.dumps(seqs))):
        assert (other.q_lens, other.kv_lens, other.total_q, other.total_kv) == ([3, 2], [4, 2], 5, 6)
        assert other.table.tolist() == seqs.table.tolist() and other.device == seqs.device
        plan, mine = _plan(other, q, k, k, True, 0.25, None), _plan(seqs, q, k, k, True, 0.25, None)
        assert plan is not mine and all(a is not b for a, b in zip(plan.tables, mine.tables))


def test_bias_after_a_move_that_failed():
    b = kb.RelativeBias(3, 8, 16, device="meta")
    with pytest.raises(NotImplementedError):
        b.to("cpu")  # the weight has nothing to copy
    assert b.buckets.is_meta
    assert b.to_empty(device="cpu").buckets.tolist() == relative_buckets(8, 16, True)
