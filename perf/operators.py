"""Timed cases of the transformer-block operators: attention over packed
sequences, the learned relative position bias inside it, its single-token form
over a cache, and the residual norm that joins two blocks.

Each case is a dict of plain values.  ``prepare`` makes the tensors a program
holds before the call, ``run`` makes one pass: with ``own`` the framework's
entry points, otherwise elementary torch operations in 32 bits.  ``exact`` is
the definition in 64 bits.
"""

import math
import random

import torch

own = False

BF16, F32 = "bf16", "f32"
_DTYPES = {BF16: torch.bfloat16, F32: torch.float32}
NUM_BUCKETS, MAX_DISTANCE, EPS = 32, 128, 1e-6
DEVICE = "cuda"


def _attention(name, heads, kv_heads, dim, dtype, n_seq, lo, hi, *, causal, bias, train, past=0, lens_seed=0):
    return {"name": name, "op": "attention", "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "n_seq": n_seq, "len_lo": lo, "len_hi": hi, "past": past, "causal": causal, "bias": bias, "train": train,
            "lens_seed": lens_seed}


def _decode(name, heads, kv_heads, dim, dtype, batch, capacity, lo, hi, *, bias, lens_seed=0):
    return {"name": name, "op": "decode", "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "n_seq": batch, "capacity": capacity, "len_lo": lo, "len_hi": hi, "bias": bias, "lens_seed": lens_seed}


def _norm(name, rows, width, dtype, kind, *, gate, branch_norm, scale, train):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "kind": kind, "gate": gate,
            "branch_norm": branch_norm, "scale": scale, "train": train}


def listed():
    return [
        # image patches: every sequence 14 x 14 patches and a class token, both directions, learned bias, a training step
        _attention("patches_bias_train", 12, 12, 64, BF16, 64, 197, 197, causal=False, bias=True, train=True),
        # text at the width of the GR-KAN feed-forward workload (32 x 1024 tokens x 768), causal, learned bias
        _attention("text_bias_train", 12, 12, 64, BF16, 32, 1024, 1024, causal=True, bias=True, train=True),
        # documents of different lengths packed into one batch, grouped heads
        _attention("packed_train", 12, 4, 64, BF16, 16, 17, 2000, causal=True, bias=False, train=True, lens_seed=1),
        # one long document, an odd length, wide heads
        _attention("long_train", 16, 4, 128, BF16, 1, 8191, 8191, causal=True, bias=False, train=True),
        # a small float32 model with an odd head width: numerics work, short sequences
        _attention("short_f32_train", 5, 5, 40, F32, 6, 1, 300, causal=False, bias=True, train=True, lens_seed=2),
        # serving: a chunk of new tokens behind a long past, no gradients
        _attention("chunk_infer", 32, 8, 128, BF16, 4, 129, 129, past=3000, causal=True, bias=False, train=False),
        # serving: one user, one token, a short cache; latency counts
        _decode("token_one", 12, 12, 64, BF16, 1, 1024, 700, 700, bias=True),
        # serving: a batch of users with caches from one token to long ones
        _decode("token_batch", 32, 8, 128, BF16, 48, 8192, 1, 8192, bias=False, lens_seed=3),
        # serving a float32 model
        _decode("token_f32", 5, 5, 40, F32, 7, 640, 1, 600, bias=True, lens_seed=4),
        # the norm between two blocks while serving a few tokens
        _norm("norm_tokens", 3, 768, BF16, "layer", gate="channel", branch_norm=False, scale=1.0, train=False),
        # and in training at the feed-forward workload's size
        _norm("norm_train", 32768, 768, BF16, "layer", gate="channel", branch_norm=True, scale=1.0, train=True),
        # a wide float32 residual stream, root-mean-square norms, a gate for each token
        _norm("norm_wide_train", 8192, 4096, F32, "rms", gate="token", branch_norm=True, scale=0.7, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["attention", "attention", "decode", "norm"])
    dtype = rng.choice([BF16, BF16, F32])
    if op == "norm":
        case = _norm("", _log_int(rng, 1, 40000), _log_int(rng, 33, 6000), dtype, rng.choice(["layer", "rms"]),
                     gate=rng.choice(["none", "channel", "token"]), branch_norm=rng.random() < 0.6,
                     scale=rng.choice([1.0, 0.7, 1.3]), train=rng.random() < 0.7)
        if rng.random() < 0.7:
            case["width"] = max(64, case["width"] // 64 * 64)
        return case
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
    dim = rng.choice([24, 40, 64, 64, 64, 80, 96, 128, 128, 128])
    bias = rng.random() < 0.4
    lens_seed = rng.randrange(1 << 30)
    if op == "decode":
        capacity = _log_int(rng, 16, 16384)
        return _decode("", heads, kv_heads, dim, dtype, _log_int(rng, 1, 96), capacity, 1, capacity, bias=bias,
                       lens_seed=lens_seed)
    hi = _log_int(rng, 1, 8192 if dtype == BF16 else 2048)
    lo = rng.choice([1, hi, max(1, hi // 3)])
    train = rng.random() < 0.7
    past = 0 if train or rng.random() < 0.5 else _log_int(rng, 1, 4096)
    return _attention("", heads, kv_heads, dim, dtype, _log_int(rng, 1, 64), lo, hi, past=past,
                      causal=rng.random() < 0.7, bias=bias, train=train, lens_seed=lens_seed)


# What a drawn case may cost: the largest listed one of its operator.
_MOST = {"attention": ("flops", "long_train"), "decode": ("bytes", "token_batch"), "norm": ("bytes", "norm_wide_train")}


def draw(rng):
    by_name = {c["name"]: c for c in listed()}
    while True:
        case = _draw_once(rng)
        key, name = _MOST[case["op"]]
        w = work(case)
        # float32 attention has a quarter of the rate at best, so a quarter of the work
        if w[key] * (4 if case["op"] == "attention" and case["dtype"] == F32 else 1) <= work(by_name[name])[key]:
            del case["name"]
            return case


def _lengths(case):
    rng = random.Random(case["lens_seed"])
    return [rng.randint(case["len_lo"], case["len_hi"]) for _ in range(case["n_seq"])]


def _visible(lq, lk, causal):
    """Pairs (query, key) that attend; causal queries are the last lq of the lk positions."""
    if not causal:
        return lq * lk
    return sum(max(0, min(lk, i + 1 + lk - lq)) for i in range(lq))


def work(case):
    size = 2 if case["dtype"] == BF16 else 4
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        mat = rows * width * size
        fwd = 4 + (case["gate"] == "token")  # x, branch (, gate) in; sum, norm out
        passes, flops = fwd, 20
        if case["train"]:
            # the two output gradients in, the gradients of x, the branch (and the gate) out
            passes, flops = fwd + 4 + (case["gate"] == "token"), 60
        return {"bytes": passes * mat, "flops": flops * rows * width}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    lens = _lengths(case)
    if case["op"] == "decode":
        keys = sum(lens)
        return {"bytes": (2 * keys * kv_heads + 2 * len(lens) * heads) * dim * size, "flops": 4 * keys * heads * dim}
    tq, tk = sum(lens), sum(lens) + len(lens) * case["past"]
    pairs = sum(_visible(n, n + case["past"], case["causal"]) for n in lens)
    q_bytes, kv_bytes = tq * heads * dim * size, tk * kv_heads * dim * size
    if not case["train"]:
        return {"bytes": 2 * q_bytes + 2 * kv_bytes, "flops": 4 * pairs * heads * dim}
    # q, k, v, the output's gradient in; the output and three gradients out
    return {"bytes": 4 * q_bytes + 4 * kv_bytes, "flops": 14 * pairs * heads * dim}


# --- inputs -------------------------------------------------------------------


def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=DEVICE) * scale).to(dtype)


def _inputs(case, seed):
    """The tensors of a case, without gradients or plans."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        t = {"x": _randn(gen, rows, width, dtype=dtype, scale=2.0) + 0.25, "branch": _randn(gen, rows, width, dtype=dtype)}
        t["weight"] = (1.0 + 0.2 * _randn(gen, width)).to(dtype)
        t["shift"] = _randn(gen, width, scale=0.1).to(dtype) if case["kind"] == "layer" else None
        t["branch_weight"] = (1.0 + 0.2 * _randn(gen, width)).to(dtype) if case["branch_norm"] else None
        t["branch_shift"] = (_randn(gen, width, scale=0.1).to(dtype)
                             if case["branch_norm"] and case["kind"] == "layer" else None)
        t["gate"] = None
        if case["gate"] == "channel":
            t["gate"] = _randn(gen, width, scale=0.5).to(dtype)
        elif case["gate"] == "token":
            t["gate"] = torch.sigmoid(_randn(gen, rows, width)).to(dtype)
        if case["train"]:
            t["d_sum"], t["d_norm"] = _randn(gen, rows, width, dtype=dtype), _randn(gen, rows, width, dtype=dtype)
        return t
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    lens = _lengths(case)
    table = _randn(gen, NUM_BUCKETS, heads, scale=0.5, dtype=dtype) if case["bias"] else None
    if case["op"] == "decode":
        n, cap = case["n_seq"], case["capacity"]
        return {"q": _randn(gen, n, heads, dim, dtype=dtype), "k": _randn(gen, n, cap, kv_heads, dim, dtype=dtype),
                "v": _randn(gen, n, cap, kv_heads, dim, dtype=dtype), "table": table, "lengths": lens}
    tq, tk = sum(lens), sum(lens) + len(lens) * case["past"]
    if case["past"]:
        q = _randn(gen, tq, heads, dim, dtype=dtype)
        k, v = _randn(gen, tk, kv_heads, dim, dtype=dtype), _randn(gen, tk, kv_heads, dim, dtype=dtype)
    else:
        # q, k and v as views of one projection's output
        qkv = _randn(gen, tq, heads + 2 * kv_heads, dim, dtype=dtype)
        q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
    t = {"q": q, "k": k, "v": v, "table": table, "lengths": lens}
    if case["train"]:
        t["d_out"] = _randn(gen, tq, heads, dim, dtype=dtype)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "t": t}
    leaves = ([k for k in ("x", "branch", "weight", "shift", "branch_weight", "branch_shift", "gate")]
              if case["op"] == "norm" else ["q", "k", "v"])
    if case["op"] == "decode":
        t["positions"] = torch.tensor(t["lengths"], dtype=torch.int32, device=DEVICE)
    if case["op"] != "norm" and case["bias"]:
        if own:
            import kanforge_b200 as kb

            state["bias"] = kb.RelativeBias(case["heads"], num_buckets=NUM_BUCKETS, max_distance=MAX_DISTANCE,
                                            bidirectional=_both_ways(case), device=DEVICE,
                                            dtype=t["table"].dtype)
            with torch.no_grad():
                state["bias"].weight.copy_(t["table"])
            if not case.get("train"):
                state["bias"].requires_grad_(False)
        # bucket of every key position minus query position that occurs
        span = max(t["lengths"]) + case.get("past", 0)
        state["buckets"] = torch.tensor([_bucket(d, _both_ways(case)) for d in range(-span, span + 1)], device=DEVICE)
        state["span"] = span
    if own and case["op"] == "attention":
        import kanforge_b200 as kb

        state["sequences"] = kb.PackedSequences(t["lengths"], [n + case["past"] for n in t["lengths"]], device=DEVICE)
    if case.get("train"):
        for name in leaves:
            if t[name] is not None:
                t[name] = t[name].requires_grad_()
        state["leaves"] = [t[name] for name in leaves if t[name] is not None]
    return state


# --- one pass -------------------------------------------------------------------


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import kanforge_b200 as kb

    case, t = state["case"], state["t"]
    if case["op"] == "decode":
        return kb.attention_decode(t["q"], t["k"], t["v"], t["positions"], bias=state.get("bias"))
    if case["op"] == "attention":
        bias = state.get("bias")
        out = kb.attention(t["q"], t["k"], t["v"], state["sequences"], causal=case["causal"], bias=bias)
        if not case["train"]:
            return out
        leaves = state["leaves"] + ([bias.weight] if bias is not None else [])
        return [out.detach(), *torch.autograd.grad(out, leaves, t["d_out"])]
    total, normed = kb.residual_norm(t["x"], t["branch"], t["weight"], t["shift"], kind=case["kind"], gate=t["gate"],
                                     branch_norm=case["branch_norm"], branch_weight=t["branch_weight"],
                                     branch_bias=t["branch_shift"], residual_scale=case["scale"], eps=EPS)
    if not case["train"]:
        return [total, normed]
    grads = torch.autograd.grad([total, normed], state["leaves"], [t["d_sum"], t["d_norm"]])
    return [total.detach(), normed.detach(), *grads]


def _run_plain(state):
    case = state["case"]
    with torch.no_grad():
        if case["op"] == "attention":
            return _plain_attention(state)
        if case["op"] == "decode":
            return _plain_decode(state)
        return _plain_norm(state)


def _both_ways(case):
    return not case.get("causal", True)


def _bucket(rel, both_ways):
    """Bucket of key position minus query position: one bucket for each small
    distance, then buckets whose edges grow geometrically up to MAX_DISTANCE.
    Exact: the logarithm's floor is taken by comparing integers."""
    n, first = NUM_BUCKETS, 0
    if both_ways:
        n //= 2
        first = n if rel > 0 else 0
        dist = abs(rel)
    else:
        dist = max(0, -rel)
    exact = n // 2
    if dist < exact:
        return first + dist
    steps = n - exact
    # the largest b < steps with dist >= exact * (MAX_DISTANCE / exact) ** (b / steps)
    b = 0
    while b + 1 < steps and dist ** steps >= exact ** (steps - b - 1) * MAX_DISTANCE ** (b + 1):
        b += 1
    return first + exact + b


def _groups(lens, past):
    """Runs of neighbouring sequences of one length: (count, length, first query row, first key row)."""
    runs, q0, k0 = [], 0, 0
    for n in lens:
        if runs and runs[-1][1] == n:
            runs[-1][0] += 1
        else:
            runs.append([1, n, q0, k0])
        q0, k0 = q0 + n, k0 + n + past
    return runs


def _plain_attention(state):
    case, t = state["case"], state["t"]
    heads, kv_heads, dim, past = case["heads"], case["kv_heads"], case["dim"], case["past"]
    rep, scale = heads // kv_heads, 1.0 / math.sqrt(dim)
    dtype = t["q"].dtype
    out = torch.empty(t["q"].shape, device=DEVICE, dtype=dtype)
    train = case["train"]
    if train:
        dq, dk, dv = (torch.empty(t[n].shape, device=DEVICE, dtype=dtype) for n in ("q", "k", "v"))
        d_table = torch.zeros(NUM_BUCKETS, heads, device=DEVICE) if case["bias"] else None

    def split(x, first, n, length, h):  # (n, kv_heads, h per kv head, length, dim)
        return x[first:first + n * length].float().reshape(n, length, kv_heads, h, dim).permute(0, 2, 3, 1, 4)

    def merge(x, n, length, h):
        return x.permute(0, 3, 1, 2, 4).reshape(n * length, kv_heads * h, dim).to(dtype)

    for n, lq, q0, k0 in _groups(t["lengths"], past):
        lk = lq + past
        q, k, v = split(t["q"], q0, n, lq, rep), split(t["k"], k0, n, lk, 1), split(t["v"], k0, n, lk, 1)
        s = (q * scale) @ k.transpose(-1, -2)
        rel = torch.arange(lk, device=DEVICE)[None, :] - (torch.arange(lq, device=DEVICE)[:, None] + past)
        if case["bias"]:
            buckets = state["buckets"][rel + state["span"]]
            s += t["table"].float().t().reshape(kv_heads, rep, NUM_BUCKETS)[:, :, buckets]
        if case["causal"]:
            s = s.masked_fill(rel > 0, -math.inf)
        p = (s - s.amax(-1, keepdim=True)).exp_()
        p /= p.sum(-1, keepdim=True)
        o = p @ v
        out[q0:q0 + n * lq] = merge(o, n, lq, rep)
        if not train:
            continue
        g = split(t["d_out"], q0, n, lq, rep)
        ds = g @ v.transpose(-1, -2)
        ds -= (g * o).sum(-1, keepdim=True)
        ds *= p
        dv[k0:k0 + n * lk] = merge((p.transpose(-1, -2) @ g).sum(2, keepdim=True), n, lk, 1)
        dk[k0:k0 + n * lk] = merge((ds.transpose(-1, -2) @ q).sum(2, keepdim=True) * scale, n, lk, 1)
        dq[q0:q0 + n * lq] = merge(ds @ k * scale, n, lq, rep)
        if case["bias"]:
            d_table.index_add_(0, buckets.flatten(), ds.sum(0).reshape(heads, lq * lk).t())
    if not train:
        return out
    return [out, dq, dk, dv] + ([d_table.to(dtype)] if case["bias"] else [])


def _plain_decode(state):
    case, t = state["case"], state["t"]
    heads, kv_heads, dim, n, cap = case["heads"], case["kv_heads"], case["dim"], case["n_seq"], case["capacity"]
    q = t["q"].float().reshape(n, kv_heads, heads // kv_heads, dim) / math.sqrt(dim)
    k, v = t["k"].float().permute(0, 2, 1, 3), t["v"].float().permute(0, 2, 1, 3)
    s = q @ k.transpose(-1, -2)
    rel = torch.arange(cap, device=DEVICE)[None, :] - (t["positions"][:, None] - 1)
    if case["bias"]:
        buckets = state["buckets"][rel.clamp(-state["span"], state["span"]) + state["span"]]
        s += t["table"].float()[buckets].permute(0, 2, 1).reshape(n, kv_heads, heads // kv_heads, cap)
    s = s.masked_fill((rel > 0)[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True)).exp_()
    return ((p @ v) / p.sum(-1, keepdim=True)).reshape(n, heads, dim).to(t["q"].dtype)


def _plain_norm(state):
    case, t = state["case"], state["t"]
    f = {k: (None if x is None else x.float()) for k, x in t.items()}
    layer, dtype = case["kind"] == "layer", t["x"].dtype

    def normed(x):
        if layer:
            x = x - x.mean(-1, keepdim=True)
        r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
        return x * r, r

    def normed_grad(g, hat, r):
        mean = g.mean(-1, keepdim=True) if layer else 0.0
        return (g - mean - hat * (g * hat).mean(-1, keepdim=True)) * r

    u = f["branch"]
    if case["branch_norm"]:
        b_hat, b_r = normed(u)
        u = b_hat * f["branch_weight"]
        if layer:
            u = u + f["branch_shift"]
    gate = f["gate"]
    total = case["scale"] * f["x"] + (u if gate is None else gate * u)
    hat, r = normed(total)
    h = hat * f["weight"]
    if layer:
        h = h + f["shift"]
    outs = [total.to(dtype), h.to(dtype)]
    if not case["train"]:
        return outs
    g = f["d_sum"] + normed_grad(f["d_norm"] * f["weight"], hat, r)
    dx = case["scale"] * g
    d_weight = (f["d_norm"] * hat).sum(0)
    du = g if gate is None else g * gate
    d_branch, grads = du, {}
    if case["branch_norm"]:
        d_branch = normed_grad(du * f["branch_weight"], b_hat, b_r)
        grads["branch_weight"] = (du * b_hat).sum(0)
        if layer:
            grads["branch_shift"] = du.sum(0)
    if layer:
        grads["shift"] = f["d_norm"].sum(0)
    if gate is not None:
        grads["gate"] = g * u if case["gate"] == "token" else (g * u).sum(0)
    grads.update(x=dx, branch=d_branch, weight=d_weight)
    order = ("x", "branch", "weight", "shift", "branch_weight", "branch_shift", "gate")
    return outs + [grads[k].to(dtype) for k in order if k in grads]


# --- the definition in 64 bits --------------------------------------------------


def exact(case, seed):
    if case["op"] == "norm" and case["rows"] * case["width"] > 1 << 26:
        return None
    t = {k: (x.double() if isinstance(x, torch.Tensor) else x) for k, x in _inputs(case, seed).items()}
    if case["op"] == "norm":
        return _exact_norm(case, t)
    return _exact_attention(case, t)


def _edge_buckets(both_ways):
    """Distances at which a new bucket begins, by the definition: bucket number
    exact + floor(log(d / exact) / log(MAX_DISTANCE / exact) * steps), at most the last one."""
    n = NUM_BUCKETS // 2 if both_ways else NUM_BUCKETS
    small = n // 2
    edges = list(range(1, small + 1))
    for b in range(1, n - small):
        d = small
        while d ** (n - small) < small ** (n - small - b) * MAX_DISTANCE ** b:
            d += 1
        edges.append(d)
    return torch.tensor(edges, device=DEVICE)


def _exact_attention(case, t):
    decode = case["op"] == "decode"
    heads, rep, dim = case["heads"], case["heads"] // case["kv_heads"], case["dim"]
    train, causal = case.get("train", False), case.get("causal", True)
    q_all = t["q"]
    out = torch.zeros_like(q_all)
    if train:
        dq, dk, dv = torch.zeros_like(q_all), torch.zeros_like(t["k"]), torch.zeros_like(t["v"])
        d_table = torch.zeros(NUM_BUCKETS, heads, dtype=torch.float64, device=DEVICE)
    both = _both_ways(case)
    edges = _edge_buckets(both)
    q0 = k0 = 0
    for b, n in enumerate(t["lengths"]):
        lq, lk = (1, n) if decode else (n, n + case["past"])
        i = torch.arange(lk - lq, lk, device=DEVICE)[:, None]
        j = torch.arange(lk, device=DEVICE)[None, :]
        if case["bias"]:
            dist = (i - j).abs() if both else (i - j).clamp(min=0)
            where = torch.bucketize(dist, edges, right=True) + ((j > i) * (NUM_BUCKETS // 2) if both else 0)
        for h in range(heads):
            if decode:
                q, k, v = q_all[b:b + 1, h], t["k"][b, :n, h // rep], t["v"][b, :n, h // rep]
            else:
                q, k, v = q_all[q0:q0 + lq, h], t["k"][k0:k0 + lk, h // rep], t["v"][k0:k0 + lk, h // rep]
            s = q @ k.T / dim ** 0.5
            if case["bias"]:
                s = s + t["table"][:, h][where]
            if causal:
                s = torch.where(j <= i, s, -math.inf)
            e = torch.exp(s - s.max(1, keepdim=True).values)
            p = e / e.sum(1, keepdim=True)
            o = p @ v
            if decode:
                out[b, h] = o[0]
                continue
            out[q0:q0 + lq, h] = o
            if not train:
                continue
            g = t["d_out"][q0:q0 + lq, h]
            ds = p * (g @ v.T - (g * o).sum(1, keepdim=True))
            dv[k0:k0 + lk, h // rep] += p.T @ g
            dk[k0:k0 + lk, h // rep] += ds.T @ q / dim ** 0.5
            dq[q0:q0 + lq, h] = ds @ k / dim ** 0.5
            if case["bias"]:
                for c in range(NUM_BUCKETS):
                    d_table[c, h] += ds[where == c].sum()
        q0, k0 = q0 + lq, k0 + lk
    if not train:
        return out
    return [out, dq, dk, dv] + ([d_table] if case["bias"] else [])


def _exact_norm(case, t):
    layer, width = case["kind"] == "layer", case["width"]

    def stats(x):
        m = x.sum(1, keepdim=True) / width if layer else torch.zeros_like(x[:, :1])
        return m, ((x - m) ** 2).sum(1, keepdim=True) / width + EPS

    leaves = {k: t[k].requires_grad_() for k in ("x", "branch", "weight", "shift", "branch_weight", "branch_shift", "gate")
              if t[k] is not None}
    u = leaves["branch"]
    if case["branch_norm"]:
        m, var = stats(u)
        u = (u - m) / var.sqrt() * leaves["branch_weight"] + leaves.get("branch_shift", 0.0)
    total = case["scale"] * leaves["x"] + leaves.get("gate", 1.0) * u
    m, var = stats(total)
    h = (total - m) / var.sqrt() * leaves["weight"] + leaves.get("shift", 0.0)
    if not case["train"]:
        return [total.detach(), h.detach()]
    grads = torch.autograd.grad((total * t["d_sum"]).sum() + (h * t["d_norm"]).sum(), list(leaves.values()))
    return [total.detach(), h.detach(), *grads]
