"""The recurrent and the local attention operators as they are measured: the gated delta rule
over whole sequences and token by token over its state, and attention with a sliding
window and first tokens that stay visible, over whole sequences and token by token
over a ring cache.

A case is a dict:
  op        "delta"        gated_delta_attention, from q, k, v, g, beta and a state
            "delta_step"   gated_delta_step: `seq` tokens, the state updated in place
            "window"       window_attention
            "window_step"  window_attention_step: one token, written into the ring cache
  dtype     of q, k, v, out, beta and the caches (g and the state are float32)
  backward  whether the call is followed by its backward for upstream gradients of all
            outputs: a training step's share, all gradients requested
  batch, q_heads, k_heads, v_heads (window: k_heads == v_heads), seq, dim
  window, sinks   of the window operators; prompt: tokens seen before a window_step

``run`` computes plain torch operations unless ``own`` is set, and the framework's
operators then.
"""

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BLOCK = 64  # tokens of a chunk of the plain delta rule


def _case(name, op, batch, heads, seq, *, dim=64, dtype="bf16", backward=False, window=0, sinks=0, prompt=0):
    q_heads, k_heads, v_heads = heads
    return dict(name=name, op=op, batch=batch, q_heads=q_heads, k_heads=k_heads, v_heads=v_heads, seq=seq, dim=dim,
                dtype=dtype, backward=backward, window=window, sinks=sinks, prompt=prompt)


def listed():
    return [
        # fine-tuning on ordinary texts, the model's heads: a length that fills no chunk, a state for two KV heads
        _case("delta_train_2x1000", "delta", 2, (14, 2, 2), 1000, backward=True),
        # the headline benchmark's batch and length, a state for every head
        _case("delta_train_4x4096", "delta", 4, (14, 14, 14), 4096, backward=True),
        # a long prompt read in once, queries and keys shared by pairs of value heads
        _case("delta_prefill_32768", "delta", 1, (7, 7, 14), 32768),
        # a short call in fp32, narrower heads: checking a layer
        _case("delta_train_2x200_fp32", "delta", 2, (8, 4, 8), 200, dim=48, dtype="fp32", backward=True),
        # answering one user: one token, a state for every head
        _case("delta_step_1", "delta_step", 1, (14, 14, 14), 1),
        # answering many users at once
        _case("delta_step_256", "delta_step", 256, (14, 14, 14), 1),
        # fine-tuning on ordinary texts with a short window
        _case("window_train_2x1000", "window", 2, (14, 2, 2), 1000, backward=True, window=256, sinks=4),
        # the headline benchmark's batch and length
        _case("window_train_4x4096", "window", 4, (14, 2, 2), 4096, backward=True, window=1024, sinks=4),
        # a long prompt read in once
        _case("window_prefill_32768", "window", 1, (14, 2, 2), 32768, window=4096, sinks=4),
        # checking a layer in fp32, narrower heads with their own KV head each
        _case("window_train_2x333_fp32", "window", 2, (8, 8, 8), 333, dim=48, dtype="fp32", backward=True, window=100, sinks=1),
        # answering one user with a full window behind
        _case("window_step_1", "window_step", 1, (14, 2, 2), 1, window=1024, sinks=4, prompt=5000),
        # answering many users, prompts of many lengths
        _case("window_step_128", "window_step", 128, (14, 2, 2), 1, window=4096, sinks=4, prompt=8192),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges."""
    op = rng.choice(["delta", "delta", "window", "window", "delta_step", "window_step"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32", "fp16"])
    dim = rng.choice([64, 64, 64, 48, 32])
    window = sinks = prompt = 0
    if op.startswith("delta"):
        heads = rng.choice([(14, 14, 14), (14, 2, 2), (7, 7, 14), (2, 2, 14), (8, 4, 8), (4, 4, 4), (1, 1, 1)])
    else:
        heads = rng.choice([(14, 2, 2), (14, 2, 2), (8, 2, 2), (4, 4, 4), (8, 1, 1), (1, 1, 1)])
        window, sinks = _spread(rng, 2, 4096), rng.choice([0, 1, 4, 4, 16, 70])
    backward = False
    if op.endswith("step"):
        batch, seq = _spread(rng, 1, 128), rng.choice([1, 1, 2, 5]) if op == "delta_step" else 1
        prompt = _spread(rng, 1, 8192) if op == "window_step" else 0
    else:
        backward = rng.random() < 0.6
        # a softmax over one token alone has gradients of zero for q and k: two at least
        seq = _spread(rng, 2 if op == "window" else 1, 8192 if dtype == "bf16" else 2048)
        batch = rng.choice([1, 1, 2, 3, 4])
        most = 56 * 4096 if dtype == "bf16" else 14 * 2048
        while batch > 1 and batch * max(heads) * seq > most:
            batch -= 1
        if backward:
            window = min(window, 1024)
    return dict(op=op, batch=batch, q_heads=heads[0], k_heads=heads[1], v_heads=heads[2], seq=seq, dim=dim, dtype=dtype,
                backward=backward, window=window, sinks=sinks, prompt=prompt)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _out_heads(case):
    return max(case["q_heads"], case["v_heads"])


def _tensors(case, seed):
    """q and k of length one for the delta rule, as its layers normalise them, and
    N(0, 1) for the softmax; decays from slow to fast over the heads."""
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    b, hq, hk, hv, n, d = (case[x] for x in ("batch", "q_heads", "k_heads", "v_heads", "seq", "dim"))

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    s = dict(case=case, scale=d ** -0.5)
    q, k, v = normal(b, hq, n, d), normal(b, hk, n, d), normal(b, hv, n, d)
    if case["op"].startswith("delta"):
        q, k = (t / (t.square().sum(-1, keepdim=True) + 1e-6).sqrt() for t in (q, k))
        rate = torch.exp(normal(hv).clamp(-2, 2) - 2)[None, :, None]
        s["g"] = -rate * torch.log1p(torch.exp(normal(b, hv, n)))
        s["beta"] = torch.sigmoid(normal(b, hv, n)).to(dtype)
        s["state"] = 0.1 * normal(b, hv, d, d)
        s["dstate"] = 0.1 * normal(b, hv, d, d)
    s["q"], s["k"], s["v"] = q.to(dtype), k.to(dtype), v.to(dtype)
    s["dout"] = normal(b, _out_heads(case), n, d).to(dtype)
    if case["op"] == "window_step":
        size, prompt = case["sinks"] + case["window"], case["prompt"]
        # prompts from a few tokens to the longest; the caches hold what a ring of that age holds
        s["positions"] = torch.randint(max(0, prompt - 3 * prompt // 4), prompt + 1, (b,), generator=gen, device=dev)
        held = torch.minimum(s["positions"], torch.full_like(s["positions"], size))
        filled = (torch.arange(size, device=dev)[None] < held[:, None])[:, None, :, None]
        s["k_cache"] = torch.where(filled, normal(b, hk, size, d), 0).to(dtype)
        s["v_cache"] = torch.where(filled, normal(b, hk, size, d), 0).to(dtype)
    return s


_WRT = {"delta": ("q", "k", "v", "g", "beta", "state"), "window": ("q", "k", "v")}


def prepare(case, seed):
    state = _tensors(case, seed)
    if case["backward"]:
        for name in _WRT[case["op"]]:
            state[name].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------


def _repeated(x, heads):
    return x if x.shape[1] == heads else x.repeat_interleave(heads // x.shape[1], 1)


def _unit_lower_inverse(a):
    """(I + a)^-1 of strictly lower a [..., C, C]: the inverses of the diagonal blocks of 1, 2, 4, ... rows."""
    c = a.shape[-1]
    at = torch.arange(c, device=a.device)
    t = torch.eye(c, device=a.device, dtype=a.dtype).expand(a.shape)
    for level in range(int(math.log2(c))):
        row, col = at[:, None] >> level, at[None, :] >> level
        below = (row == col + 1) & (row % 2 == 1)
        t = t - t @ (a * below) @ t
    return t


def _delta_plain(q, k, v, g, beta, state, scale):
    """The chunked delta rule: the chunks' maps of the state S -> M S + D combined in doubling strides."""
    b, hv, n, d = v.shape
    heads, dtype = max(q.shape[1], hv), q.dtype
    pad = -n % _BLOCK
    q, k, v, beta = (torch.nn.functional.pad(t.float(), (0, 0) * (t.ndim - 3) + (0, pad)) for t in (q, k, v, beta))
    q, k, v, beta = (t.view(*t.shape[:2], -1, _BLOCK, *t.shape[3:]) for t in (q, k, v, beta))
    k = _repeated(k, hv)
    # sums of decays in float64: differences of them are what the rule needs
    total = torch.nn.functional.pad(g.double(), (0, pad)).view(b, hv, -1, _BLOCK).cumsum(-1)
    low = torch.tril(torch.ones((_BLOCK, _BLOCK), dtype=torch.bool, device=q.device))
    decay = torch.exp(torch.where(low, total[..., :, None] - total[..., None, :], -math.inf)).float()
    since = torch.exp(total).float()[..., None]
    until = torch.exp(total[..., -1:] - total).float()[..., None]
    last = since[..., -1:, :]
    kt = k.transpose(-1, -2)
    t = _unit_lower_inverse(torch.tril(k @ kt * decay, -1) * beta[..., None, :])
    free, read = t @ v, t @ (since * k)
    write = (until * k).transpose(-1, -2)
    eye = torch.eye(d, device=q.device)
    maps, adds = last * eye - write @ (beta[..., None] * read), write @ (beta[..., None] * free)
    adds = torch.cat((maps[:, :, :1] @ state[:, :, None] + adds[:, :, :1], adds[:, :, 1:]), 2)
    chunks = maps.shape[2]
    for level in range(max(0, chunks - 1).bit_length()):
        w = 1 << level
        adds = torch.cat((adds[:, :, :w], maps[:, :, w:] @ adds[:, :, :-w] + adds[:, :, w:]), 2)
        maps = torch.cat((maps[:, :, :w], maps[:, :, w:] @ maps[:, :, :-w]), 2)
    before = torch.cat((state[:, :, None], adds[:, :, :-1]), 2)
    u = beta[..., None] * (free - read @ before)
    qh, kh, uh, sh, dh, gh = (_repeated(x, heads) for x in (q, k, u, before, decay, since))
    out = scale * (gh * qh @ sh + (qh @ kh.transpose(-1, -2) * dh) @ uh)
    return out.flatten(2, 3)[:, :, :n].to(dtype), adds[:, :, -1]


def _delta_step_plain(q, k, v, g, beta, state, scale):
    """Token by token; the state is updated in place."""
    heads, hv = max(q.shape[1], v.shape[1]), v.shape[1]
    qf, kf, vf, bf = _repeated(q.float(), heads), _repeated(k.float(), hv), v.float(), beta.float()
    s, outs = state, []
    for t in range(q.shape[2]):
        s = s * torch.exp(g[:, :, t, None, None])
        u = bf[:, :, t, None] * (vf[:, :, t] - (s * kf[:, :, t, :, None]).sum(2))
        s = s + kf[:, :, t, :, None] * u[:, :, None]
        outs.append(scale * (_repeated(s, heads) * qf[:, :, t, :, None]).sum(2))
    state.copy_(s)
    return torch.stack(outs, 2).to(q.dtype), state


def _window_plain(q, k, v, window, sinks, scale):
    """Blocks of queries over the keys of their windows, beside the first keys where the window has left them."""
    b, hq, n, d = q.shape
    hk, dtype, dev = k.shape[1], q.dtype, q.device
    size = max(16, min(128, window))
    pad = -n % size
    blocks = (n + pad) // size
    qf = torch.nn.functional.pad(q.float() * scale, (0, 0, 0, pad)).view(b, hk, hq // hk, blocks, size, d)
    kf, vf = (torch.nn.functional.pad(t.float(), (0, 0, window - 1, pad)) for t in (k, v))
    kw, vw = (t.unfold(2, window - 1 + size, size)[:, :, None] for t in (kf, vf))  # [b, hk, 1, blocks, d, span]
    row = torch.arange(blocks, device=dev)[:, None, None] * size + torch.arange(size, device=dev)[:, None]
    col = torch.arange(blocks, device=dev)[:, None, None] * size + torch.arange(window - 1 + size, device=dev) - (window - 1)
    near = (col >= 0) & (col <= row) & (row - col < window) & (col < n)
    far = row - torch.arange(min(sinks, n), device=dev) >= window
    score = torch.where(near, qf @ kw, -math.inf)
    first = torch.where(far, qf @ k[:, :, :sinks].float().transpose(-1, -2)[:, :, None, None], -math.inf)
    score = torch.cat((first, score), -1)
    score = torch.where(row < n, score, 0.0)
    p = torch.exp(score - score.detach().amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    far_part, near_part = p[..., :far.shape[-1]], p[..., far.shape[-1]:]
    out = near_part @ vw.transpose(-1, -2) + far_part @ v[:, :, :sinks].float()[:, :, None, None]
    return out.reshape(b, hq, blocks * size, d)[:, :, :n].to(dtype)


def _window_step_plain(q, k, v, k_cache, v_cache, positions, window, sinks, scale):
    b, hq, _, d = q.shape
    hk, at = k.shape[1], torch.arange(b, device=q.device)
    slot = torch.where(positions < sinks, positions, sinks + (positions - sinks) % window)
    k_cache[at, :, slot] = k[:, :, 0]
    v_cache[at, :, slot] = v[:, :, 0]
    size = sinks + window
    filled = torch.arange(size, device=q.device)[None] <= torch.clamp(positions, max=size - 1)[:, None]
    score = scale * (q.float().view(b, hk, hq // hk, d) @ k_cache.float().transpose(-1, -2))
    score = torch.where(filled[:, None, None], score, -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p / p.sum(-1, keepdim=True)) @ v_cache.float()
    return out.view(b, hq, 1, d).to(q.dtype), k_cache, v_cache


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _call(s):
    """(outputs of the operator as a tuple)"""
    case = s["case"]
    op, window = case["op"], dict(window=case["window"], sinks=case["sinks"], scale=s["scale"])
    if own:
        if op == "delta":
            from oal_amd.gated_delta import gated_delta_attention

            return gated_delta_attention(s["q"], s["k"], s["v"], s["g"], s["beta"], scale=s["scale"], initial_state=s["state"])
        if op == "delta_step":
            from oal_amd.gated_delta import gated_delta_step

            return gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], scale=s["scale"]), s["state"]
        if op == "window":
            from oal_amd.window_attention import window_attention

            return (window_attention(s["q"], s["k"], s["v"], **window),)
        from oal_amd.window_attention import window_attention_step

        out = window_attention_step(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["positions"], **window)
        return out, s["k_cache"], s["v_cache"]
    if op == "delta":
        return _delta_plain(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["scale"])
    if op == "delta_step":
        return _delta_step_plain(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["scale"])
    if op == "window":
        return (_window_plain(s["q"], s["k"], s["v"], **window),)
    return _window_step_plain(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["positions"], **window)


def run(state):
    case = state["case"]
    if not case["backward"]:
        with torch.no_grad():
            return _call(state)
    outs = _call(state)
    upstream = (state["dout"], state["dstate"]) if case["op"] == "delta" else (state["dout"],)
    grads = torch.autograd.grad(outs, [state[x] for x in _WRT[case["op"]]], upstream)
    return tuple(t.detach() for t in outs) + tuple(grads)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def _pairs(n, window, sinks):
    """Visible pairs of n queries."""
    full = min(n, window)
    near = full * (full + 1) // 2 + (n - full) * window
    past = max(0, n - window)  # queries that have left behind 1, 2, ... first keys
    most = min(sinks, past)
    return near + most * (most + 1) // 2 + (past - most) * sinks


def work(case):
    """Each operand read once and each result written once. The delta rule: the state's
    read, its update and the queries' reads, token by token; attention: the two products over visible pairs."""
    b, hq, hk, hv, n, d = (case[x] for x in ("batch", "q_heads", "k_heads", "v_heads", "seq", "dim"))
    size, heads = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]], _out_heads(case)
    ins, outs = b * n * d * (hq + hk + hv) * size, b * n * d * heads * size
    if case["op"].startswith("delta"):
        gates, states = b * n * hv * (4 + size), 2 * b * hv * d * d * 4
        flops = b * n * d * d * (4.0 * hv + 2.0 * heads)
        if case["backward"]:
            # the inputs and dout in, out, the gradients and both states' out
            return {"bytes": 2 * ins + 2 * outs + 2 * gates + 2 * states, "flops": 3 * flops}
        return {"bytes": ins + outs + gates + states, "flops": flops}
    if case["op"] == "window":
        flops = 4.0 * d * b * hq * _pairs(n, case["window"], case["sinks"])
        if case["backward"]:
            return {"bytes": 2 * ins + 2 * outs, "flops": 3.5 * flops}
        return {"bytes": ins + outs, "flops": flops}
    # positions run from a quarter of the prompt to all of it
    seen = min(case["sinks"] + case["window"], case["prompt"] * 5 // 8 + 1)
    return {"bytes": ins + outs + b * 8 + 2 * b * hk * (seen + 1) * d * size, "flops": 4.0 * b * hq * seen * d}


# ---------------------------------------------------------------------------
# The same from the definition in 64 bits
# ---------------------------------------------------------------------------


def _exact_delta(s):
    """The recurrence over tokens, and its reverse."""
    case, scale = s["case"], s["scale"]
    b, n, d, hv = (case[x] for x in ("batch", "seq", "dim", "v_heads"))
    heads, hq, hk = _out_heads(case), case["q_heads"], case["k_heads"]
    each = heads // hv  # output heads of a state
    q = s["q"].detach().double().repeat_interleave(heads // hq, 1).view(b, hv, each, n, d)
    k = s["k"].detach().double().repeat_interleave(hv // hk, 1)
    v, g, beta, state = (s[x].detach().double() for x in ("v", "g", "beta", "state"))
    past, written, read, out = [], [], [], []
    for t in range(n):
        past.append(state if case["backward"] else None)
        kept = state * g[:, :, t, None, None].exp()
        r = v[:, :, t] - (kept.transpose(-1, -2) @ k[:, :, t, :, None])[..., 0]
        u = beta[:, :, t, None] * r
        state = kept + k[:, :, t, :, None] * u[:, :, None, :]
        out.append(scale * q[:, :, :, t] @ state)
        read.append(r)
        written.append(u)
    final = state
    out = torch.stack(out, 3).reshape(b, heads, n, d)
    if case["op"] == "delta_step" or not case["backward"]:
        return out, final
    do = s["dout"].double().view(b, hv, each, n, d)
    ds = s["dstate"].double()
    dq, dk, dv, dg, dbeta = [], [], [], [], []
    for t in range(n - 1, -1, -1):
        kept = past[t] * g[:, :, t, None, None].exp()
        kt, u, r = k[:, :, t], written[t], read[t]
        now = kept + kt[..., None] * u[:, :, None, :]
        dq.append(scale * do[:, :, :, t] @ now.transpose(-1, -2))
        ds = ds + scale * q[:, :, :, t].transpose(-1, -2).contiguous() @ do[:, :, :, t]
        du = (ds.transpose(-1, -2) @ kt[..., None])[..., 0]
        dr = beta[:, :, t, None] * du
        dbeta.append((du * r).sum(-1))
        dv.append(dr)
        dk.append((ds @ u[..., None])[..., 0] - (kept @ dr[..., None])[..., 0])
        dkept = ds - kt[..., None] * dr[:, :, None, :]
        dg.append((dkept * kept).sum((-1, -2)))
        ds = dkept * g[:, :, t, None, None].exp()
    dq = torch.stack(dq[::-1], 3).reshape(b, hq, heads // hq, n, d).sum(2)
    dk = torch.stack(dk[::-1], 2).view(b, hk, hv // hk, n, d).sum(2)
    dv, dg, dbeta = (torch.stack(t[::-1], 2) for t in (dv, dg, dbeta))
    return out, final, dq, dk, dv, dg, dbeta, ds


def _exact_window(s):
    """Rows of queries, each over all keys that it sees."""
    case, scale = s["case"], s["scale"]
    b, hq, hk, n, d = (case[x] for x in ("batch", "q_heads", "k_heads", "seq", "dim"))
    window, sinks, r = case["window"], case["sinks"], hq // hk
    q, k, v, do = (s[x].detach().double() for x in ("q", "k", "v", "dout"))
    out, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    at = torch.arange(n, device=q.device)
    rows = max(16, min(n, 2048))
    for h in range(hq):
        for i0 in range(0, n, rows):
            i1 = min(n, i0 + rows)
            keep = at[:i1][(at[:i1] < sinks) | (at[:i1] > i0 - window)]
            i = at[i0:i1, None]
            seen = (keep <= i) & ((i - keep < window) | (keep < sinks))
            for x in range(b):
                kk, vv, qq, dd = k[x, h // r, keep], v[x, h // r, keep], q[x, h, i0:i1], do[x, h, i0:i1]
                p = torch.softmax((scale * qq @ kk.T).masked_fill(~seen, -math.inf), -1)
                out[x, h, i0:i1] = p @ vv
                if case["backward"]:
                    dp = dd @ vv.T
                    dscore = scale * p * (dp - (p * dp).sum(-1, keepdim=True))
                    dq[x, h, i0:i1] = dscore @ kk
                    dk[x, h // r, keep] += dscore.T @ qq
                    dv[x, h // r, keep] += p.T @ dd
    return (out, dq, dk, dv) if case["backward"] else (out,)


def _exact_window_step(s):
    case = s["case"]
    b, hq, hk, d = (case[x] for x in ("batch", "q_heads", "k_heads", "dim"))
    window, sinks = case["window"], case["sinks"]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    out = torch.empty((b, hq, 1, d), dtype=torch.float64, device=kc.device)
    for x, p in enumerate(s["positions"].tolist()):
        slot = p if p < sinks else sinks + (p - sinks) % window
        kc[x, :, slot], vc[x, :, slot] = s["k"][x, :, 0].double(), s["v"][x, :, 0].double()
        count = min(p + 1, sinks + window)
        kk, vv = (t[x, :, :count].repeat_interleave(hq // hk, 0) for t in (kc, vc))
        weight = torch.softmax(s["scale"] * (s["q"][x].double() * kk).sum(-1), -1)
        out[x, :, 0] = (weight[..., None] * vv).sum(1)
    return out, kc, vc


def exact(case, seed):
    if case["op"].startswith("delta"):
        # every state is kept for the reverse
        if case["batch"] * case["v_heads"] * case["seq"] * case["dim"] ** 2 * 8 > 4e10:
            return None
        return _exact_delta(_tensors(case, seed))
    return _exact_window(_tensors(case, seed)) if case["op"] == "window" else _exact_window_step(_tensors(case, seed))
