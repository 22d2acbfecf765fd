"""The operators of a transformer block's forward pass, as cases that can be measured.

    fc_bf16_residual   C = R + s * act(A . Wp^T + bias)
    norm_residual      t = R + s * gate * norm(x);  y = norm(t)
    attention_bf16     softmax(scale * q . k^T) . v over packed sequences, grouped heads, causal or full

`run` computes a case in its plain form (elementary torch operations in 32 bits) or, with `own` set, by the
calls a user makes.  `exact` restates the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

BF16, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------ cases
# Widths 4096 and 1000 are the wide MLP's of this repository's benchmark; 128 and 64 are the usual head widths.

def _fc(m, n, k, act, bias=True, residual="", scale=1.0, out="bf16", **kw):
    return dict(op="fc", m=m, n=n, k=k, act=act, bias=bias, residual=residual, scale=scale, out=out, **kw)


def _norm(rows, d, x="bf16", residual="bf16", sum="bf16", y="bf16", post="", pre="rms", gate="", gate_rows=0, scale=1.0, **kw):
    return dict(op="norm", rows=rows, d=d, x=x, residual=residual, sum=sum, y=y, post=post, pre=pre, gate=gate,
                gate_rows=gate_rows, scale=scale, **kw)


def _prompt(batch, longest, ragged, hq, hkv, d, causal, **kw):
    return dict(op="prompt", batch=batch, longest=longest, ragged=ragged, hq=hq, hkv=hkv, d=d, causal=causal, **kw)


def _token(batch, capacity, ragged, new, hq, hkv, d, **kw):
    return dict(op="token", batch=batch, capacity=capacity, ragged=ragged, new=new, hq=hq, hkv=hkv, d=d, **kw)


def listed():
    return [
        # one new token through the output projection of an attention block
        _fc(1, 4096, 4096, "none", residual="bf16", name="fc_token"),
        # a ragged batch of rows into a narrow odd width, fp32 residual stream
        _fc(777, 1000, 4096, "gelu", residual="f32", scale=0.5, out="f32", name="fc_ragged"),
        # a prompt batch through a whole layer: product, bias, activation, residual
        _fc(16384, 4096, 4096, "gelu_tanh", residual="bf16", name="fc_prompt"),
        # the norm before a block for one new token
        _norm(1, 4096, name="norm_token"),
        # images with a gate of their own each (197 rows an image), odd width, fp32 stream, layer norm
        _norm(788, 1000, residual="f32", sum="f32", pre="layer", gate="f32", gate_rows=197, name="norm_gated"),
        # a prompt batch with norms on both sides of the block
        _norm(8192, 4096, post="rms", pre="rms", scale=0.7, name="norm_both"),
        # the largest batch of the benchmark's width: fp32 stream, one gate vector for all rows
        _norm(65536, 4096, residual="f32", sum="f32", pre="layer", gate="f32", name="norm_large"),
        # serving: one new token each for 64 sequences with caches of very different lengths
        _token(64, 4096, True, 1, 32, 8, 128, name="attention_tokens"),
        # serving one user far into a long text
        _token(1, 65536, False, 1, 32, 8, 128, name="attention_long_cache"),
        # a packed batch of prompts of different lengths
        _prompt(16, 2048, True, 32, 8, 128, True, name="attention_packed"),
        # one long prompt
        _prompt(1, 16384, False, 16, 4, 128, True, name="attention_prompt"),
        # image patches: full attention, one key head for each query head, 64 wide, a length that is no multiple of a tile
        _prompt(64, 197, False, 16, 16, 64, False, name="attention_images"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["fc", "norm", "prompt", "token"])
    dt = lambda: rng.choice(["bf16", "f32"])
    if op == "fc":
        n, k = _log(rng, 40, 8192), 8 * _log(rng, 8, 1024)
        if rng.random() < 0.5:
            n = max(8, n // 8 * 8)
        top = 16384 * 4096 * 4096 // (n * k)
        m = _log(rng, 1, max(1, min(16384, top)))
        return _fc(m, n, k, rng.choice(["none", "relu", "tanh", "gelu", "gelu_tanh", "silu"]), rng.random() < 0.7,
                   rng.choice(["", "bf16", "f32"]), rng.choice([1.0, 0.5, 0.3]), dt())
    if op == "norm":
        d = _log(rng, 40, 8192)
        if rng.random() < 0.6:
            d = max(8, d // 8 * 8)
        rows = _log(rng, 1, min(65536, 65536 * 4096 // d))
        gate = rng.choice(["", "bf16", "f32"])
        return _norm(rows, d, dt(), rng.choice(["", "bf16", "f32"]), dt(), dt(), rng.choice(["", "rms", "layer"]),
                     rng.choice(["rms", "layer"]), gate, rng.choice([0, 1, _log(rng, 1, rows)]) if gate else 0,
                     rng.choice([1.0, 0.25]))
    hkv = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 5, 7, 8])
    d = rng.choice([64, 128, 128, 72, 96, 40])
    if op == "prompt":
        longest = _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(64, (8192 // longest) ** 2, 16384 // longest)))
        while hkv * g > 16:
            g = max(1, g // 2)
        return _prompt(batch, longest, rng.random() < 0.6, hkv * g, hkv, d, rng.random() < 0.7)
    capacity = _log(rng, 1, 65536)
    batch = _log(rng, 1, max(1, min(128, 262144 // capacity)))
    return _token(batch, capacity, rng.random() < 0.6, rng.choice([1, 1, 1, 2, 4]) if capacity >= 8 else 1, hkv * g, hkv, d)


# ------------------------------------------------------------------ inputs

def _dt(name):
    return {"bf16": BF16, "f32": F32}[name]


def _lengths(case):
    """Host list: the sequences' lengths (prompts) or their caches' filled lengths (tokens); part of the case, as any size is."""
    r = np.random.default_rng([case["batch"], case["hq"], case["d"]])
    top = case["longest"] if case["op"] == "prompt" else case["capacity"]
    low = 1 if case["op"] == "prompt" else case["new"]
    if not case["ragged"]:
        return [top] * case["batch"]
    n = np.exp(r.uniform(math.log(max(low, top / 16)), math.log(top + 1), case["batch"]))
    return [int(min(top, max(low, v))) for v in n]


def _offsets(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32), device="cuda")


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *shape, dtype=F32, s=1.0: (torch.randn(shape, generator=g, device="cuda", dtype=F32) * s).to(dtype)
    if case["op"] == "fc":
        m, n, k = case["m"], case["n"], case["k"]
        return dict(a=rn(m, k, dtype=BF16), wp=rn(n, k, dtype=BF16, s=k ** -0.5), bias=rn(n, s=0.2) if case["bias"] else None,
                    residual=rn(m, n, dtype=_dt(case["residual"]), s=2.0) if case["residual"] else None)
    if case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        t = dict(x=rn(rows, d, dtype=_dt(case["x"])),
                 residual=rn(rows, d, dtype=_dt(case["residual"]), s=3.0) if case["residual"] else None, gate=None)
        if case["gate"]:
            count = 1 if case["gate_rows"] == 0 else -(-rows // case["gate_rows"])
            t["gate"] = rn(count, d, dtype=_dt(case["gate"]), s=0.5)
        for side in ("post", "pre"):
            kind = case[side]
            t[side] = (kind, 1.0 + rn(d, s=0.1), rn(d, s=0.1) if kind == "layer" else None, 1e-5) if kind else None
        return t
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    n = _lengths(case)
    if case["op"] == "prompt":
        # q, k and v are what one projection wrote: columns of one tensor of packed rows
        t = rn(sum(n), (hq + 2 * hkv) * d, dtype=BF16)
        q, k, v = t.split((hq * d, hkv * d, hkv * d), dim=1)
        view = lambda x, h: x.unflatten(1, (h, d))
        off = _offsets(n)
        return dict(q=view(q, hq), k=view(k, hkv), v=view(v, hkv), n_q=n, n_k=n, off_q=off, off_k=off, start=None, k_lens=None)
    batch, cap, new = case["batch"], case["capacity"], case["new"]
    q = rn(batch * new, hq, d, dtype=BF16)
    k, v = rn(batch * cap, hkv, d, dtype=BF16), rn(batch * cap, hkv, d, dtype=BF16)
    return dict(q=q, k=k, v=v, n_q=[new] * batch, n_k=n, off_q=_offsets([new] * batch), off_k=_offsets([cap] * batch),
                k_lens=torch.tensor(n, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own:
        import swcompiler_b200 as swc
        state["be"] = swc.Backend(torch.cuda.current_device(), swc.TC_BF16)
    return state


# ------------------------------------------------------------------ one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    import swcompiler_b200 as swc
    case, be = s["case"], s["be"]
    if case["op"] == "fc":
        act = {"none": swc.ACT_NONE, "relu": swc.ACT_RELU, "tanh": swc.ACT_TANH, "gelu": swc.ACT_GELU,
               "gelu_tanh": swc.ACT_GELU_TANH, "silu": swc.ACT_SILU}[case["act"]]
        return be.fc_bf16_residual(s["a"], s["wp"], s["bias"], act, residual=s["residual"], scale=case["scale"],
                                   out_dtype=_dt(case["out"]))
    if case["op"] == "norm":
        kind = {"rms": swc.NORM_RMS, "layer": swc.NORM_LAYER}
        post, pre = [(kind[p[0]],) + p[1:] if p else None for p in (s["post"], s["pre"])]
        return be.norm_residual(s["x"], residual=s["residual"], post=post, gate=s["gate"], gate_rows=case["gate_rows"],
                                scale=case["scale"], pre=pre, sum_dtype=_dt(case["sum"]), y_dtype=_dt(case["y"]))
    return be.attention_bf16(s["q"], s["k"], s["v"], s["off_q"], s["off_k"], k_lens=s["k_lens"],
                             causal=case.get("causal", True))


def _plain_norm(t, p):
    kind, weight, bias, eps = p
    if kind == "layer":
        t = t - t.mean(1, keepdim=True)
    t = t * torch.rsqrt((t * t).mean(1, keepdim=True) + eps) * weight
    return t if bias is None else t + bias


def _plain_act(t, act):
    if act == "relu":
        return torch.clamp_min(t, 0)
    if act == "tanh":
        return torch.tanh(t)
    if act == "gelu":
        return 0.5 * t * torch.erfc(t * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return t / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (t + 0.044715 * t * t * t)))
    if act == "silu":
        return t / (1 + torch.exp(-t))
    return t


def _run_plain(s):
    case = s["case"]
    if case["op"] == "fc":
        t = s["a"].float() @ s["wp"].float().t()
        if s["bias"] is not None:
            t = t + s["bias"]
        t = _plain_act(t, case["act"]) * case["scale"]
        if s["residual"] is not None:
            t = s["residual"].float() + t
        return t.to(_dt(case["out"]))
    if case["op"] == "norm":
        t = s["x"].float()
        if s["post"]:
            t = _plain_norm(t, s["post"])
        t = t * case["scale"]
        if s["gate"] is not None:
            gate = s["gate"].float()
            if case["gate_rows"]:
                gate = gate[torch.arange(case["rows"], device="cuda") // case["gate_rows"]]
            t = t * gate
        if s["residual"] is not None:
            t = t + s["residual"].float()
        return t.to(_dt(case["sum"])), _plain_norm(t, s["pre"]).to(_dt(case["y"]))
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    causal = case.get("causal", True)
    out = torch.empty((s["q"].shape[0], hq, d), dtype=BF16, device="cuda")
    at_q = at_k = 0
    for b in range(case["batch"]):
        nq, nk = s["n_q"][b], s["n_k"][b]
        k = s["k"][at_k:at_k + nk].float().transpose(0, 1)              # [hkv, nk, d]
        v = s["v"][at_k:at_k + nk].float().transpose(0, 1)
        piece = max(1, min(nq, (1 << 28) // (hq * nk)))                  # scores of at most a GiB at a time
        for i in range(0, nq, piece):
            c = min(piece, nq - i)
            q = s["q"][at_q + i:at_q + i + c].float().transpose(0, 1)    # [hq, c, d]
            scores = (q.reshape(hkv, hq // hkv * c, d) @ k.transpose(1, 2)) * d ** -0.5
            if causal:
                last = torch.arange(i, i + c, device="cuda") + (nk - nq)
                hidden = torch.arange(nk, device="cuda") > last[:, None]
                scores = scores.view(hq, c, nk).masked_fill_(hidden, -math.inf).view(hkv, -1, nk)
            p = torch.exp_(scores - scores.amax(2, keepdim=True))
            o = (p @ v) / p.sum(2, keepdim=True)
            out[at_q + i:at_q + i + c] = o.view(hq, c, d).transpose(0, 1)
        at_q += nq
        at_k += nk if case["op"] == "prompt" else case["capacity"]
    return out


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    w = lambda t: None if t is None else t.double()
    if case["op"] == "fc":
        t = torch.einsum("mk,nk->mn", w(s["a"]), w(s["wp"]))
        if s["bias"] is not None:
            t += w(s["bias"])
        act = case["act"]
        if act == "relu":
            t = torch.where(t > 0, t, torch.zeros_like(t))
        elif act == "tanh":
            t = torch.tanh(t)
        elif act == "gelu":
            t = t * torch.special.ndtr(t)
        elif act == "gelu_tanh":
            t = 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3)))
        elif act == "silu":
            t = t * torch.sigmoid(t)
        return t * case["scale"] + (w(s["residual"]) if s["residual"] is not None else 0)
    if case["op"] == "norm":
        outs = ([], [])
        rows, step = case["rows"], max(1, (1 << 25) // case["d"])

        def norm(t, p):
            kind, weight, bias, eps = p
            if kind == "layer":
                var, mean = torch.var_mean(t, dim=1, correction=0, keepdim=True)
                return (t - mean) / torch.sqrt(var + eps) * w(weight) + w(bias)
            return t / torch.sqrt(t.square().sum(1, keepdim=True) / t.shape[1] + eps) * w(weight)

        for i in range(0, rows, step):
            j = min(rows, i + step)
            t = w(s["x"][i:j])
            if s["post"]:
                t = norm(t, s["post"])
            if s["gate"] is not None:
                every = case["gate_rows"] or rows
                t = t * w(s["gate"])[[r // every for r in range(i, j)]]
            t = t * case["scale"] + (w(s["residual"][i:j]) if s["residual"] is not None else 0)
            outs[0].append(t)
            outs[1].append(norm(t, s["pre"]))
        return torch.cat(outs[0]), torch.cat(outs[1])
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    out = torch.zeros((s["q"].shape[0], hq, d), dtype=torch.float64, device="cuda")
    first_q, first_k = s["off_q"].tolist(), s["off_k"].tolist()
    for b, (nq, nk) in enumerate(zip(s["n_q"], s["n_k"])):
        for h in range(hq):
            k = w(s["k"][first_k[b]:first_k[b] + nk, h // (hq // hkv)])
            v = w(s["v"][first_k[b]:first_k[b] + nk, h // (hq // hkv)])
            step = max(1, (1 << 27) // nk)
            for i in range(0, nq, step):
                j = min(nq, i + step)
                z = torch.einsum("id,jd->ij", w(s["q"][first_q[b] + i:first_q[b] + j, h]), k) / math.sqrt(d)
                if case.get("causal", True):
                    seen = torch.ones((j - i, nk), dtype=torch.bool, device="cuda").tril(i + nk - nq)
                    z = torch.where(seen, z, -math.inf)
                out[first_q[b] + i:first_q[b] + j, h] = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) @ v
    return out


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    size = {"": 0, "bf16": 2, "f32": 4}
    if case["op"] == "fc":
        m, n, k = case["m"], case["n"], case["k"]
        return dict(bytes=2 * m * k + 2 * n * k + 4 * n * case["bias"] + m * n * (size[case["residual"]] + size[case["out"]]),
                    flops=2 * m * n * k)
    if case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        gates = 0 if not case["gate"] else 1 if case["gate_rows"] == 0 else -(-rows // case["gate_rows"])
        vectors = sum({"": 0, "rms": 1, "layer": 2}[case[side]] for side in ("post", "pre"))
        return dict(bytes=rows * d * (size[case["x"]] + size[case["residual"]] + size[case["sum"]] + size[case["y"]]) +
                    gates * d * size[case["gate"]] + 4 * d * vectors,
                    flops=rows * d * (4 + 6 * bool(case["post"]) + 6))
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    n_k = _lengths(case)
    n_q = n_k if case["op"] == "prompt" else [case["new"]] * case["batch"]
    pairs = sum(q * k - (q * (q - 1) // 2 if case.get("causal", True) else 0) for q, k in zip(n_q, n_k))
    return dict(bytes=2 * d * (2 * hq * sum(n_q) + 2 * hkv * sum(n_k)), flops=4 * hq * d * pairs)
