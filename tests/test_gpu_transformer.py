"""The KAN transformer on the GPU: training against the same stack in 64 bits,
and tokens one at a time over a cache against whole sequences.

Tolerances are fractions of the compared tensor's largest magnitude.  Each of
the some twenty operators on a path here is right to about 1e-6 (float32) or
2^-8 of it (bfloat16, one rounding of its output) and none amplifies more than
a few times: 1e-4 and 0.1.
"""

from __future__ import annotations

import math

import pytest
import torch

import kanforge_b200 as kb

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.float32: 1e-4, torch.bfloat16: 0.1}


def close(got, want, tol):
    want = want.double()
    assert got.shape == want.shape
    assert (got.double() - want).abs().max() <= tol * want.abs().max().clamp_min(1e-30)


def model(dtype=torch.float32, causal=True, seed=0, **kw):
    torch.manual_seed(seed)
    m = kb.KANTransformer(48, 2, 6, 2, 64, causal=causal, num_buckets=8, max_distance=20, groups=8, **kw)
    with torch.no_grad():
        for p in (m.bias.weight, *(b.attention_norm.gate for b in m.blocks if b.attention_norm.gate is not None)):
            p.copy_(torch.randn_like(p) * 0.5)
    return m.to(device=DEV, dtype=dtype)


def plain_norm(n, y):
    y = y - y.mean(-1, keepdim=True) if n.kind == "layer" else y
    return y * torch.rsqrt(y.square().mean(-1, keepdim=True) + n.eps)


def affine(v, w, b):
    return v * w.double() + (0.0 if b is None else b.double())


def plain_join(n, x, branch):
    if branch is None:
        return x, affine(plain_norm(n, x), n.weight, n.bias)
    u = affine(plain_norm(n, branch), n.branch_weight, n.branch_bias) if n.branch_norm else branch
    y = n.residual_scale * x + (u if n.gate is None else n.gate.double() * u)
    return y, affine(plain_norm(n, y), n.weight, n.bias)


def plain(m, x, lens):
    """The stack in float64, but for the KAN layers (float32, as they are)."""
    x, h = plain_join(m.start, x, None)
    for b in m.blocks:
        q, k, v = (h @ b.qkv.weight.double().T).unflatten(-1, (-1, b.head_dim)).split([b.heads, b.kv_heads, b.kv_heads], dim=-2)
        k, v = (t.repeat_interleave(b.heads // b.kv_heads, dim=-2) for t in (k, v))
        out, at = [], 0
        for n in lens:
            s = slice(at, at + n)
            at += n
            t = torch.einsum("qhd,khd->hqk", q[s], k[s]) / math.sqrt(b.head_dim)
            i = torch.arange(n, device=DEV)
            dist = i[:, None] - i[None, :]
            t = t + m.bias.weight.double()[m.bias.buckets[dist.clamp(-20, 20) + 20].long()].permute(2, 0, 1)
            if m.causal:
                t = t.masked_fill(dist < 0, -math.inf)
            out.append(torch.einsum("hqk,khd->qhd", t.softmax(-1), v[s]))
        x, h = plain_join(b.attention_norm, x, torch.cat(out).flatten(-2) @ b.proj.weight.double().T)
        x, h = plain_join(b.ffn_norm, x, b.ffn(h.float()).double())
    return h


@pytest.mark.parametrize("causal,kw", [(True, {}), (False, dict(norm="rms", branch_norm=True, gate_init=1.0)),
                                       (True, dict(kind="kan", gate_init=0.5))])
def test_training_step_against_64_bits(causal, kw):
    m = model(causal=causal, **kw)
    lens = [1, 40, 0, 131, 7]
    x = torch.randn(sum(lens), 48, device=DEV, requires_grad=True)
    g = torch.randn_like(x)
    seqs = kb.PackedSequences(lens, device=DEV)
    params = list(m.parameters())
    h = m(x, seqs)
    got = torch.autograd.grad((h * g).sum(), [x, *params])
    ref = plain(m, x.double(), lens)
    want = torch.autograd.grad((ref * g.double()).sum(), [x, *params])
    close(h, ref.detach(), TOL[torch.float32])
    for a, b in zip(got, want):
        close(a, b, TOL[torch.float32])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_over_a_cache_follow_the_whole_sequences(dtype):
    m = model(dtype, gate_init=1.0)
    lens, new = [5, 33, 1, 0], 6
    total = [n + new for n in lens]
    rows = [torch.randn(n, 48, device=DEV, dtype=dtype) for n in total]
    with torch.no_grad():
        whole = m(torch.cat(rows), kb.PackedSequences(total, device=DEV)).split(total)
    cache = m.new_cache(len(lens), 40)
    prompt = m.prefill(torch.cat([r[:n] for r, n in zip(rows, lens)]), lens, cache).split(lens)
    for p, w, n in zip(prompt, whole, lens):
        if n:
            close(p, w[:n], TOL[dtype])
    for t in range(new):
        h = m.decode(torch.stack([r[n + t] for r, n in zip(rows, lens)]), cache)
        close(h, torch.stack([w[n + t] for w, n in zip(whole, lens)]), TOL[dtype])
    assert cache.lengths.tolist() == total and cache.longest == 39
    m.decode(torch.zeros(4, 48, device=DEV, dtype=dtype), cache)
    with pytest.raises(ValueError):
        m.decode(torch.zeros(4, 48, device=DEV, dtype=dtype), cache)


def test_a_few_steps_of_training_lower_the_loss():
    m = model(torch.bfloat16, gate_init=1.0)
    lens = [64, 17, 200]
    x = torch.randn(sum(lens), 48, device=DEV, dtype=torch.bfloat16)
    want = torch.randn_like(x)
    seqs = kb.PackedSequences(lens, device=DEV)
    opt = torch.optim.SGD(m.parameters(), lr=0.05)
    losses = []
    for _ in range(8):
        opt.zero_grad()
        loss = (m(x, seqs).float() - want.float()).square().mean()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    assert all(math.isfinite(v) for v in losses) and losses[-1] < losses[0]


def test_a_decoding_step_replays_from_a_graph():
    heads, dim, capacity = 6, 64, 512
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    q, k, v = r(3, heads, dim), r(3, capacity, 2, dim), r(3, capacity, 2, dim)
    x, w = r(3, heads * dim), r(heads * dim)
    lengths = torch.tensor([1, 300, 77], dtype=torch.int32, device=DEV)

    def step():
        o = kb.attention_decode(q, k, v, lengths)
        return kb.residual_norm(x, o.flatten(1), w, kind="rms")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = step()
    for n in ([1, 300, 77], [2, 512, 0]):
        lengths.copy_(torch.tensor(n, dtype=torch.int32))
        q.copy_(r(3, heads, dim))
        graph.replay()
        for a, b in zip((y, h), step()):
            assert torch.equal(a, b)


def test_the_models_step_replays_from_a_graph_up_to_the_capacity():
    """Beyond it the sequences that are full answer NaN; the others go on."""
    m = model(torch.bfloat16, gate_init=1.0)
    lens, capacity = [5, 33, 1], 36
    rows = torch.randn(sum(lens), 48, device=DEV, dtype=torch.bfloat16)
    tokens = torch.randn(6, 3, 48, device=DEV, dtype=torch.bfloat16)
    want_cache, cache = m.new_cache(3, 64), m.new_cache(3, capacity)
    for c in (want_cache, cache):
        m.prefill(rows, lens, c)
    x = tokens[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.decode(x, cache)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h = m.decode(x, cache)
    want = [m.decode(t, want_cache) for t in tokens]
    for n in range(1, 6):
        x.copy_(tokens[n])
        graph.replay()
        full = 33 + n + 1 > capacity
        assert h[1].isnan().all() == full
        for s in (0, 2) if full else (0, 1, 2):
            close(h[s], want[n][s], TOL[torch.bfloat16])
    assert cache.lengths.tolist() == [n + 6 for n in lens]
    assert cache.longest == 34  # the prompt and the one step that ran outside the graph
