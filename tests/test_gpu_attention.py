"""Attention over packed sequences, its relative position bias and the
single-token form against the formulas in float64.

Tolerance, max|a - b| / max|b| over a tensor: bfloat16 2e-2, about ten roundings
of 2^-9 (the inputs are taken as exact; the probabilities, dS, the output that
delta is made of and the results are each rounded once).  float32 1e-5, 168
roundings of 2^-24: sums of up to 1000 terms with errors of either sign.
"""

from __future__ import annotations

import math

import pytest
import torch

import kanforge_b200 as kb
from kanforge_b200.attention import relative_buckets

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 1e-5, torch.bfloat16: 2e-2}


def close(got, want, tol, what, floor=0.0):
    assert got.shape == want.shape, what
    if got.numel() == 0:
        return
    assert got.isfinite().all(), f"{what} is not finite"
    top = max(want.abs().max().item(), floor)
    err = (got.double() - want).abs().max().item()
    assert err <= tol * max(top, 1e-30), f"{what}: {err:.3e} of {top:.3e}"


def formula(q, k, v, q_lens, kv_lens, causal, scale, table=None, buckets=None, span=0):
    """float64, differentiable; rows that see no key give 0."""
    rep = q.shape[1] // k.shape[1]
    outs, q0, k0 = [], 0, 0
    for lq, lk in zip(q_lens, kv_lens):
        qs, ks, vs = q[q0:q0 + lq], k[k0:k0 + lk].repeat_interleave(rep, 1), v[k0:k0 + lk].repeat_interleave(rep, 1)
        s = torch.einsum("ihd,jhd->hij", qs, ks) * scale
        dist = torch.arange(lq, device=q.device)[:, None] + (lk - lq) - torch.arange(lk, device=q.device)[None, :]
        if table is not None:
            s = s + table[buckets[dist.clamp(-span, span) + span].long()].permute(2, 0, 1)
        seen = (dist >= 0) if causal else torch.ones_like(dist, dtype=torch.bool)
        e = torch.where(seen, (s - s.detach().masked_fill(~seen, -1e300).amax(-1, keepdim=True) if lk else s), -1e4).exp()
        e = e * seen
        outs.append(torch.einsum("hij,jhd->ihd", e / e.sum(-1, keepdim=True).clamp(min=1e-300), vs))
        q0, k0 = q0 + lq, k0 + lk
    return torch.cat(outs) if outs else q * 0


def make(q_lens, kv_lens, heads, kv_heads, dim, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda n, h: (scale * torch.randn(n, h, dim, generator=g, device="cuda")).to(dtype)  # noqa: E731
    return r(sum(q_lens), heads), r(sum(kv_lens), kv_heads), r(sum(kv_lens), kv_heads), r(sum(q_lens), heads)


def check(q, k, v, dout, q_lens, kv_lens, causal, bias=None, scale=None, tol=None):
    dtype = q.dtype
    seqs = kb.PackedSequences(q_lens, kv_lens)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)] + ([bias.weight] if bias is not None else [])
    out = kb.attention(*leaves[:3], seqs, causal=causal, bias=bias, scale=scale)
    assert out.dtype == dtype and out.shape == q.shape
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        infer = kb.attention(q, k, v, seqs, causal=causal, bias=bias, scale=scale)
    assert torch.equal(infer, out)
    ref = [t.detach().double().requires_grad_() for t in leaves]
    want = formula(*ref[:3], q_lens, kv_lens, causal, scale or 1 / math.sqrt(q.shape[-1]), *(
        (ref[3], bias.buckets, bias.max_distance) if bias is not None else ()))
    wants = torch.autograd.grad((want * dout.double()).sum(), ref, allow_unused=True)
    tol = tol or TOL[dtype]
    close(out, want.detach(), tol, "out")
    # a sequence of one visible key has dS = 0 exactly: then compare with the size of its terms
    for name, g, w, leaf in zip(("dq", "dk", "dv", "dbias"), grads, wants, leaves):
        w = torch.zeros_like(leaf, dtype=torch.float64) if w is None else w
        close(g, w, TOL[g.dtype] if name != "dbias" else TOL[dtype], name, floor=0.1)
    return out, grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [8, 24, 40, 64, 80, 128])
def test_head_widths(dim, causal, dtype):
    lens = [70, 1, 129, 256, 33]
    check(*make(lens, lens, 4, 2, dim, dtype), lens, lens, causal)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 6), (6, 2), (8, 1), (12, 4), (20, 1), (33, 11)])
def test_shared_heads(heads, kv_heads, dtype):
    lens = [65, 200, 3]
    check(*make(lens, lens, heads, kv_heads, 64, dtype), lens, lens, True)


LAYOUTS = [
    ([1], [1]), ([0], [0]), ([], []), ([0, 5, 0], [0, 5, 0]), ([1] * 9, [1] * 9), ([64, 128, 192], [64, 128, 192]),
    ([127, 129, 255, 257], [127, 129, 255, 257]), ([600], [600]),
    ([1, 1, 1], [500, 1, 77]), ([5, 70, 130], [300, 70, 514]),  # queries behind a past
    ([10, 200, 64], [4, 130, 0]), ([150], [20]), ([3, 0], [0, 9]),  # causal rows that see nothing, no keys, no queries
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("layout", LAYOUTS, ids=lambda x: f"{x[0]}over{x[1]}")
def test_lengths(layout, causal, dtype):
    q_lens, kv_lens = layout
    out, grads = check(*make(q_lens, kv_lens, 6, 3, 64, dtype), q_lens, kv_lens, causal)
    q0 = 0
    for lq, lk in zip(q_lens, kv_lens):
        empty = lq if lk == 0 else (max(0, lq - lk) if causal else 0)
        assert (out[q0:q0 + empty] == 0).all() and (grads[0][q0:q0 + empty] == 0).all()
        q0 += lq


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("buckets,span", [(32, 128), (8, 20), (4, 3), (64, 500)])
def test_bias(buckets, span, causal, dtype):
    lens = [1, 90, 260, 300]
    heads = 6
    bias = kb.RelativeBias(heads, buckets, span, bidirectional=not causal, device="cuda", dtype=dtype)
    with torch.no_grad():
        bias.weight.normal_(0, 0.7, generator=torch.Generator(device="cuda").manual_seed(5))
    check(*make(lens, lens, heads, 3, 64, dtype), lens, lens, causal, bias=bias)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bias_behind_a_past_and_wide_heads(dtype):
    q_lens, kv_lens = [5, 140, 1], [400, 141, 700]
    bias = kb.RelativeBias(4, 32, 128, bidirectional=False, device="cuda", dtype=dtype)
    with torch.no_grad():
        bias.weight.normal_(0, 0.7, generator=torch.Generator(device="cuda").manual_seed(5))
    check(*make(q_lens, kv_lens, 4, 4, 128, dtype), q_lens, kv_lens, True, bias=bias)


def test_a_bias_that_closes_a_bucket():
    # the lowest finite value keeps keys out of the softmax wherever another key is open
    lens = [200]
    for low in (torch.finfo(torch.float32).min, -float("inf")):
        q, k, v, dout = make(lens, lens, 2, 2, 64, torch.float32)
        bias = kb.RelativeBias(2, 8, 16, bidirectional=False, device="cuda")
        with torch.no_grad():
            bias.weight[-1] = low  # distances from the last bucket's first on
        first = relative_buckets(8, 16, False)[16:].index(7)
        out = kb.attention(q, k, v, kb.PackedSequences(lens), causal=True, bias=bias)
        s = torch.einsum("ihd,jhd->hij", q.double(), k.double()) / 8
        d = torch.arange(200, device="cuda")[:, None] - torch.arange(200, device="cuda")[None, :]
        p = s.masked_fill((d < 0) | (d >= first), -math.inf).softmax(-1)
        close(out.detach(), torch.einsum("hij,jhd->ihd", p, v.double()), 1e-5, "out")
        g = torch.autograd.grad(out, bias.weight, dout)[0]
        assert g.isfinite().all() and (g[-1] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_scores(dtype):
    # one key takes nearly all the weight; sums stay finite and exact at the top.  The scores reach some hundreds:
    # float32 holds them to 2^-24 * 2^9, so the probabilities to 3e-5
    lens = [150, 40]
    q, k, v, dout = make(lens, lens, 4, 4, 64, dtype, scale=6.0)
    check(q, k, v / 6, dout / 6, lens, lens, True, tol=1e-4 if dtype == torch.float32 else None)


def test_views_of_one_projection_and_odd_alignment():
    lens = [100, 57]
    g = torch.Generator(device="cuda").manual_seed(0)
    qkv = torch.randn(157, 8 + 2 * 2, 64, generator=g, device="cuda").bfloat16()
    q, k, v = qkv.split([8, 2, 2], 1)
    seqs = kb.PackedSequences(lens)
    want = kb.attention(q.contiguous(), k.contiguous(), v.contiguous(), seqs)
    assert torch.equal(kb.attention(q, k, v, seqs), want)
    odd = torch.empty(157 * 8 * 64 + 3, device="cuda", dtype=torch.bfloat16)[3:].view(157, 8, 64).copy_(q)
    assert torch.equal(kb.attention(odd, k, v, seqs), want)
    heads_first = q.permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert torch.equal(kb.attention(heads_first, k, v, seqs), want)
    # a gradient that comes as a broadcast view
    ql = q.contiguous().requires_grad_()
    a = torch.autograd.grad(kb.attention(ql, k, v, seqs).sum(), ql)[0]
    b = torch.autograd.grad(kb.attention(ql, k, v, seqs), ql, torch.ones_like(ql))[0]
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
def test_other_sequences_never_enter(causal, dtype):
    lens = [100, 30, 77]
    q, k, v, dout = make(lens, lens, 4, 2, 64, dtype)
    seqs = kb.PackedSequences(lens)

    def step(q, k, v, dout):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = kb.attention(*leaves, seqs, causal=causal)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout)]

    want = step(q, k, v, dout)
    for t, bad in ((q, float("nan")), (k, float("inf")), (v, float("nan")), (dout, float("-inf"))):
        t[100:130] = bad
    got = step(q, k, v, dout)
    for a, b in zip(got, want):
        assert torch.equal(a[:100], b[:100]) and torch.equal(a[130:], b[130:])


def test_gradient_matches_differences():
    q_lens, kv_lens = [5, 9], [7, 6]
    q, k, v, dout = make(q_lens, kv_lens, 4, 2, 16, torch.float32)
    bias = kb.RelativeBias(4, 8, 6, bidirectional=True, device="cuda")
    with torch.no_grad():
        bias.weight.normal_(0, 0.5, generator=torch.Generator(device="cuda").manual_seed(1))
    seqs = kb.PackedSequences(q_lens, kv_lens)
    leaves = [t.requires_grad_() for t in (q, k, v)] + [bias.weight]

    def loss():
        return (kb.attention(*leaves[:3], seqs, causal=False, bias=bias).double() * dout.double()).sum()

    grads = torch.autograd.grad(loss(), leaves)
    for t, g in zip(leaves, grads):
        d = torch.randn_like(t)
        d /= d.norm()
        step = 2e-2
        with torch.no_grad():
            t += step * d
            hi = loss()
            t -= 2 * step * d
            lo = loss()
            t += step * d
        assert abs((hi - lo).item() / (2 * step) - (g.double() * d.double()).sum().item()) < 5e-3


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_same_bits_every_run_and_on_another_stream(dtype):
    lens = [400, 333, 90]
    q, k, v, dout = make(lens, lens, 8, 2, 64, dtype)
    bias = kb.RelativeBias(8, 32, 64, bidirectional=False, device="cuda", dtype=dtype)
    seqs = kb.PackedSequences(lens)

    def step():
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = kb.attention(*leaves, seqs, bias=bias)
        return [out.detach(), *torch.autograd.grad(out, leaves + [bias.weight], dout)]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    kb.kernels.check_device_errors()
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_refusals():
    q, k, v, _ = make([4], [4], 4, 2, 16, torch.float32)
    seqs = kb.PackedSequences([4])
    with pytest.raises(ValueError):
        kb.attention(q[:3], k, v, seqs)
    with pytest.raises(ValueError):
        kb.attention(q, k, v[:, :1], seqs)
    with pytest.raises(ValueError):
        kb.attention(q[:, :3], k, v, seqs)
    with pytest.raises(TypeError):
        kb.attention(q, k.bfloat16(), v, seqs)
    with pytest.raises(TypeError):
        kb.attention(q.half(), k.half(), v.half(), seqs)
    with pytest.raises(TypeError):
        kb.attention(q, k, v, [4])
    with pytest.raises(RuntimeError):
        kb.attention(q.cpu(), k.cpu(), v.cpu(), seqs)
    with pytest.raises(ValueError):
        kb.attention(q, k, v, kb.PackedSequences([4], device="cpu"))
    with pytest.raises(ValueError):
        kb.attention(q, k, v, seqs, bias=kb.RelativeBias(3, device="cuda"))
    with pytest.raises(ValueError):
        kb.attention(q, k, v, seqs, bias=kb.RelativeBias(4))
    for dim in (12, 136):
        with pytest.raises(ValueError):
            kb.attention(*make([4], [4], 4, 2, dim, torch.float32)[:3], seqs)
    q.requires_grad_()
    g = torch.autograd.grad(kb.attention(q, k, v, seqs).sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


# --- one token over a cache ---------------------------------------------------


def decode_case(batch, capacity, heads, kv_heads, dim, dtype, lengths, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    return (r(batch, heads, dim), r(batch, capacity, kv_heads, dim), r(batch, capacity, kv_heads, dim),
            torch.tensor(lengths, dtype=torch.int32, device="cuda"))


def decode_want(q, k, v, lengths, bias):
    cap = k.shape[1]
    lens = [min(max(n, 0), cap) for n in lengths]
    packed = [torch.cat([t[b, :n] for b, n in enumerate(lens)]).double() for t in (k, v)]
    return formula(q.double(), *packed, [1] * len(lens), lens, True, 1 / math.sqrt(q.shape[-1]), *(
        (bias.weight.double(), bias.buckets, bias.max_distance) if bias is not None else ()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 8), (5, 5, 40), (12, 4, 64), (8, 1, 128), (40, 2, 80), (17, 1, 64)])
def test_decode(heads, kv_heads, dim, with_bias, dtype):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 300, 511, 512, 0, 700, -3]
    q, k, v, n = decode_case(len(lengths), 512, heads, kv_heads, dim, dtype, lengths)
    bias = None
    if with_bias:
        bias = kb.RelativeBias(heads, 32, 100, bidirectional=False, device="cuda", dtype=dtype).requires_grad_(False)
        bias.weight.normal_(0, 0.7, generator=torch.Generator(device="cuda").manual_seed(5))
    got = kb.attention_decode(q, k, v, n, bias=bias)
    close(got, decode_want(q, k, v, lengths, bias), TOL[dtype], "decode")
    assert (got[11] == 0).all() and (got[13] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,capacity", [(1, 1), (1, 33), (1, 9000), (3, 4096), (200, 70)])
def test_decode_sizes(batch, capacity, dtype):
    lengths = [capacity - (b * 7) % max(1, capacity // 2) for b in range(batch)]
    q, k, v, n = decode_case(batch, capacity, 8, 2, 64, dtype, lengths)
    close(kb.attention_decode(q, k, v, n), decode_want(q, k, v, lengths, None), TOL[dtype], "decode")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_reads_no_slot_past_the_length(dtype):
    lengths = [1, 40, 129]
    q, k, v, n = decode_case(3, 130, 6, 3, 64, dtype, lengths)
    want = kb.attention_decode(q, k, v, n)
    for b, m in enumerate(lengths):
        k[b, m:], v[b, m:] = float("nan"), float("inf")
    assert torch.equal(kb.attention_decode(q, k, v, n), want)


def test_decode_cache_in_another_order():
    # (batch, kv_heads, capacity, dim) storage, viewed in the call's order
    q, k, v, n = decode_case(4, 100, 4, 2, 64, torch.bfloat16, [100, 3, 50, 77])
    kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    assert torch.equal(kb.attention_decode(q, kt, vt, n), kb.attention_decode(q, k, v, n))


def test_decode_past_32_bit_offsets():
    # the cache holds more than 2^31 elements; only the last sequence's end is looked at
    cap, kv_heads, dim = 1 << 20, 8, 128
    k = torch.zeros(3, cap, kv_heads, dim, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    q = torch.randn(3, kv_heads, dim, device="cuda").bfloat16()
    k[2, cap - 1] = q[2] * 4
    v[2, cap - 1] = torch.randn(kv_heads, dim, device="cuda").bfloat16()
    n = torch.tensor([1, 1, cap], dtype=torch.int32, device="cuda")
    got = kb.attention_decode(q, k, v, n)
    s = 4 * q[2].double().square().sum(-1, keepdim=True) / math.sqrt(dim)
    p = s.exp() / (s.exp() + cap - 1)
    assert (got[:2] == 0).all()
    close(got[2], p * v[2, cap - 1].double(), 2e-2, "last slot")


def test_decode_agrees_with_attention():
    lens = [30, 200, 77]
    q, k, v, n = decode_case(3, 256, 8, 2, 64, torch.bfloat16, lens)
    packed = [torch.cat([t[b, :m] for b, m in enumerate(lens)]) for t in (k, v)]
    want = kb.attention(q, *packed, kb.PackedSequences([1, 1, 1], lens))
    close(kb.attention_decode(q, k, v, n), want.double(), 2e-2, "decode")


def test_decode_refusals():
    q, k, v, n = decode_case(2, 8, 4, 2, 16, torch.float32, [1, 2])
    with pytest.raises(ValueError):
        kb.attention_decode(q, k, v, n.long())
    with pytest.raises(ValueError):
        kb.attention_decode(q[:1], k, v, n)
    with pytest.raises(ValueError):
        kb.attention_decode(q, k, v, n[:1])
    with pytest.raises(TypeError):
        kb.attention_decode(q, k.bfloat16(), v.bfloat16(), n)
    with pytest.raises(RuntimeError):
        kb.attention_decode(q.requires_grad_(), k, v, n)
    with pytest.raises(RuntimeError):
        kb.attention_decode(q.detach().cpu(), k.cpu(), v.cpu(), n.cpu())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (4, 1, 96), (8, 2, 64)])
def test_the_largest_bias_table(heads, kv_heads, dim, dtype):
    lens = [300, 1, 700]
    bias = kb.RelativeBias(heads, 256, 512, bidirectional=True, device="cuda", dtype=dtype)
    with torch.no_grad():
        bias.weight.normal_(0, 0.7, generator=torch.Generator(device="cuda").manual_seed(5))
    check(*make(lens, lens, heads, kv_heads, dim, dtype), lens, lens, False, bias=bias)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim", [(6, 2, 64), (4, 4, 40), (4, 1, 128), (3, 3, 104)])
@pytest.mark.parametrize("q_lens,kv_lens", [([16], [4100]), ([1], [8192]), ([70, 3], [2100, 1500]), ([300, 1, 0, 9], [1040, 30, 5, 0])])
def test_few_queries_over_many_keys(q_lens, kv_lens, heads, kv_heads, dim, causal):
    """The keys of a sequence are shared out among CTAs; short ones leave some of them none."""
    bias = kb.RelativeBias(heads, 16, 100, bidirectional=not causal, device="cuda")
    with torch.no_grad():
        bias.weight.normal_(0, 0.7, generator=torch.Generator(device="cuda").manual_seed(5))
    for b in (None, bias):
        check(*make(q_lens, kv_lens, heads, kv_heads, dim, torch.bfloat16), q_lens, kv_lens, causal, bias=b)


def test_few_queries_repeat_to_the_bit():
    q, k, v = make([40], [5000], 8, 2, 128, torch.bfloat16)[:3]
    seqs = kb.PackedSequences([40], [5000])
    first = kb.attention(q, k, v, seqs)
    for _ in range(5):
        assert torch.equal(first, kb.attention(q, k, v, seqs))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_decode_with_the_largest_bias_table(dtype):
    bias = kb.RelativeBias(32, 256, 512, bidirectional=True, device="cuda", dtype=dtype)
    with torch.no_grad():
        bias.weight.normal_(0, 0.7, generator=torch.Generator(device="cuda").manual_seed(5))
    g = torch.Generator(device="cuda").manual_seed(7)
    n = 3000
    q, k, v = (torch.randn(1, *s, generator=g, device="cuda").to(dtype) for s in ((32, 128), (4096, 2, 128), (4096, 2, 128)))
    got = kb.attention_decode(q, k, v, torch.tensor([n], dtype=torch.int32, device="cuda"), bias=bias.requires_grad_(False))
    dist = torch.arange(n - 1, -1, -1, device="cuda")
    t = torch.einsum("hd,khd->hk", q[0].double(), k[0, :n].double().repeat_interleave(16, 1)) / 128**0.5
    t = t + bias(dist).double().T
    want = torch.einsum("hk,khd->hd", t.softmax(-1), v[0, :n].double().repeat_interleave(16, 1))
    # float32: sums over 128 and 3000 terms; bfloat16: one rounding of the output
    assert (got[0].double() - want).abs().max() <= (1e-5 if dtype == torch.float32 else 2.0**-8) * want.abs().max()


@pytest.mark.parametrize("dim", [64, 80, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("layout", [([150], [20]), ([300], [0]), ([400], [30]), ([700, 300, 20], [130, 0, 20])], ids=lambda x: f"{x[0]}over{x[1]}")
def test_row_tiles_without_keys(layout, causal, dim):
    """Whole tiles of queries that see no key, beside tiles that do: exactly 0, and no gradient."""
    q_lens, kv_lens = layout
    out, grads = check(*make(q_lens, kv_lens, 8, 2, dim, torch.bfloat16), q_lens, kv_lens, causal)
    q0 = 0
    for lq, lk in zip(q_lens, kv_lens):
        empty = lq if lk == 0 else (max(0, lq - lk) if causal else 0)
        assert (out[q0:q0 + empty] == 0).all() and (grads[0][q0:q0 + empty] == 0).all()
        q0 += lq


@pytest.mark.parametrize("heads,kv_heads,dim,lens", [(2, 1, 128, [2048]), (1, 1, 128, [2048]), (1, 1, 64, [2048]), (2, 1, 128, [2048, 100]),
                                                     (1, 1, 64, [2048, 100])])
def test_slices_of_the_keys_without_work(heads, kv_heads, dim, lens):
    """Keys shared out among CTAs where full row tiles leave whole slices without a key, without a bias: the right
    values, and the same bits every time."""
    q, k, v, dout = make(lens, lens, heads, kv_heads, dim, torch.bfloat16)
    out, _ = check(q, k, v, dout, lens, lens, True)
    seqs = kb.PackedSequences(lens)
    with torch.no_grad():
        for _ in range(50):
            assert torch.equal(kb.attention(q, k, v, seqs), out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensors_in_another_layout(dtype):
    """Views of one projection that come back contiguous, from the host or from any other hook."""
    lens = [100, 57]
    qkv = torch.randn(157, 8, 64, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(dtype).requires_grad_()
    seqs = kb.PackedSequences(lens)
    grads = []
    for hooks in (torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t), torch.autograd.graph.save_on_cpu(),
                  torch.autograd.graph.saved_tensors_hooks(lambda t: t.transpose(0, -1).contiguous(), lambda t: t.transpose(0, -1))):
        with hooks:
            out = kb.attention(*qkv.split([4, 2, 2], 1), seqs)
        grads.append(torch.autograd.grad(out.float().square().sum(), qkv)[0])
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_bias_whose_tensors_were_put_in_place_one_by_one(dtype):
    lens = [40, 90]
    q, k, v, dout = make(lens, lens, 4, 2, 64, dtype)
    whole = kb.RelativeBias(4, 8, 20, bidirectional=False, device="cuda", dtype=dtype)
    with torch.no_grad():
        whole.weight.normal_(0, 0.7, generator=torch.Generator(device="cuda").manual_seed(5))
    moved = kb.RelativeBias(4, 8, 20, bidirectional=False)  # the buckets stay on the host
    moved.weight = torch.nn.Parameter(whole.weight.detach().clone())
    emptied = kb.RelativeBias(4, 8, 20, bidirectional=False, device="meta").to_empty(device="cuda").to(dtype)
    emptied.load_state_dict(whole.state_dict())
    cache = [t[:100].reshape(2, 50, 2, 64).contiguous() for t in (k, v)]
    n = torch.tensor([50, 33], dtype=torch.int32, device="cuda")
    want = None
    for b in (whole, moved, emptied):
        out, grads = check(q, k, v, dout, lens, lens, True, bias=b)
        with torch.no_grad():
            got = [out, *grads, kb.attention_decode(q[:2], *cache, n, bias=b)]
        want = want or got
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_buckets_outside_the_table_count_as_the_nearest(dtype):
    lens = [40, 90]
    q, k, v, _ = make(lens, lens, 4, 2, 64, dtype)
    bias = kb.RelativeBias(4, 8, 20, bidirectional=False, device="cuda", dtype=dtype).requires_grad_(False)
    bias.weight.normal_(0, 0.7, generator=torch.Generator(device="cuda").manual_seed(5))
    cache = [t[:100].reshape(2, 50, 2, 64).contiguous() for t in (k, v)]
    n = torch.tensor([50, 33], dtype=torch.int32, device="cuda")

    def run():
        return kb.attention(q, k, v, kb.PackedSequences(lens), bias=bias), kb.attention_decode(q[:2], *cache, n, bias=bias)

    near = bias.buckets.clone()
    near[25:27], near[30:] = 0, 7
    far = near.clone()
    far[25], far[26], far[30:] = -1, -(1 << 31), (1 << 31) - 1
    bias.buckets.copy_(near)
    want = run()
    bias.buckets.copy_(far)
    assert all(torch.equal(x, y) for x, y in zip(run(), want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (4, 1, 128)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("closed", ["a head", "the first distances", "a head but for the far ones"])
def test_biases_of_the_lowest_value(closed, causal, heads, kv_heads, dim, dtype):
    """Rows whose keys all have the type's lowest value as a bias: their scores round to it (in 64 bits, too), so
    every key weighs the same, forward and backward, near and far."""
    lens = [1, 2, 90, 400]
    bias = kb.RelativeBias(heads, 16, 40, bidirectional=not causal, device="cuda", dtype=dtype)
    low = torch.finfo(dtype).min
    with torch.no_grad():
        bias.weight.normal_(0, 0.7, generator=torch.Generator(device="cuda").manual_seed(5))
        if closed == "the first distances":
            bias.weight[:3] = low
        else:
            bias.weight[:, 1] = low
        if closed == "a head but for the far ones":
            bias.weight[7, 1] = bias.weight[15, 1] = 0.5
    check(*make(lens, lens, heads, kv_heads, dim, dtype), lens, lens, causal, bias=bias)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low", [-1e4, -1e9, -1e30])
def test_weights_add_up_to_one_under_any_mask_value(low, dtype):
    """sum over keys of dV = sum over queries of dO, whatever the rounding of the scores: each row's weights add up
    to 1 in the backward as in the forward.  bfloat16: each dV is rounded once (2^-9) and the weights are (2^-9);
    float32: P loses 2^-13 by a score of 1e4 that product and bias round to."""
    lens = [300]
    q, k, v, dout = make(lens, lens, 4, 2, 64, dtype)
    bias = kb.RelativeBias(4, 16, 40, bidirectional=False, device="cuda")
    with torch.no_grad():
        bias.weight.fill_(low)
    v.requires_grad_()
    out = kb.attention(q, k, v, kb.PackedSequences(lens), bias=bias)
    dv = torch.autograd.grad(out, v, dout)[0].double()
    terms = dout.double().reshape(300, 2, 2, 64).sum(2)
    err = (dv.sum(0) - terms.sum(0)).abs().max()
    assert err <= (2.0**-8 if dtype == torch.bfloat16 else 2.0**-12) * terms.abs().sum(0).max()
    assert (out[0].double() - v[0].double().repeat_interleave(2, 0)).abs().max() <= 2.0**-8 * v.abs().max()


def derivative_calls():
    """(name, function, inputs) of calls that need no gradient."""
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    seqs, w = kb.PackedSequences([5, 3]), r(32)
    n = torch.tensor([4, 7], dtype=torch.int32, device="cuda")
    return [("attention", lambda q, k, v: kb.attention(q, k, v, seqs), (r(8, 4, 16), r(8, 2, 16), r(8, 2, 16))),
            ("attention_decode", lambda q, k, v: kb.attention_decode(q, k, v, n), (r(2, 4, 16), r(2, 9, 2, 16), r(2, 9, 2, 16))),
            ("residual_norm", lambda x, b: kb.residual_norm(x, b, w, kind="rms")[1], (r(6, 32), r(6, 32))),
            ("first norm", lambda x: kb.residual_norm(x, None, w, kind="rms")[1], (r(6, 32),))]


@pytest.mark.parametrize("i", range(4))
def test_forward_mode_derivatives_are_refused_not_dropped(i):
    from torch.autograd import forward_ad

    _, f, args = derivative_calls()[i]
    want = f(*args)
    for j in range(len(args)):
        with forward_ad.dual_level():
            assert torch.equal(f(*args), want)  # no input carries a tangent
            dual = [forward_ad.make_dual(a, torch.ones_like(a)) if k == j else a for k, a in enumerate(args)]
            with pytest.raises(NotImplementedError):
                f(*dual)
            with torch.no_grad(), pytest.raises(NotImplementedError):
                f(*dual)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("i", range(4))
def test_a_traced_call_computes(i):
    _, f, args = derivative_calls()[i]
    with torch.no_grad():
        traced = torch.jit.trace(f, args, check_trace=False)
        other = [a * 0.5 + 0.25 for a in args]
        for a in (args, other):
            assert torch.equal(traced(*a), f(*a))


def test_tables_outlive_the_calls_that_read_them_on_another_stream():
    q = torch.randn(347, 2, 64, device="cuda")
    seqs = kb.PackedSequences([300, 40, 7])
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(first):
        want = kb.attention(q, q, q, seqs)
    tables = {t.data_ptr() for t in seqs._tiles.values()}
    torch.cuda.synchronize()
    with torch.cuda.stream(second):
        torch.cuda._sleep(1_500_000_000)  # some 0.8 s
        got = kb.attention(q, q, q, seqs)
    del seqs
    with torch.cuda.stream(first):
        new = [torch.empty(8, 8, dtype=torch.int32, device="cuda") for _ in range(64)]
    assert not second.query(), "the call was over too soon to tell"
    assert not tables & {t.data_ptr() for t in new}
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows_with_odd_strides(dtype):
    """Tensors without elements count as contiguous whatever their strides."""
    full = torch.randn(3, 2, 19, device="cuda").to(dtype)[..., 2:18]
    none = torch.randn(0, 2, 19, device="cuda").to(dtype)[..., 2:18]
    for q, kv, lens in ((full, none, ([3], [0])), (none, full, ([0], [3]))):
        leaves = [t.detach().requires_grad_() for t in (q, kv, kv)]
        out = kb.attention(*leaves, kb.PackedSequences(*lens))
        assert out.shape == q.shape and not out.any()
        assert not any(g.any() for g in torch.autograd.grad(out, leaves, torch.ones_like(out)))
    cache = torch.randn(3, 0, 2, 19, device="cuda").to(dtype)[..., 2:18]
    assert not kb.attention_decode(full, cache, cache, torch.ones(3, dtype=torch.int32, device="cuda")).any()
