"""The token mixers of long-sequence language models: what is measured of them.

Attention with a sliding window and a few first tokens that stay visible ("window"), and linear attention with a
decay for each head ("decay"), each as a prompt, as single tokens on what earlier tokens left, and as a training
step.  Everything is FP32, as every tensor of this repository.  Where `own` is true the calls go to the library, else
the same is computed with elementary torch operations.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------- cases

def window_case(name, mode, n, heads, kv_heads, q_len, kv_len, head_dim, window, sinks, ragged, head_inner=True):
    c = dict(op="window", mode=mode, n=n, heads=heads, kv_heads=kv_heads, q_len=q_len, kv_len=kv_len, head_dim=head_dim,
             window=window, sinks=sinks, ragged=ragged, head_inner=head_inner)
    return dict(c, name=name) if name else c


def decay_case(name, mode, n, heads, length, key_dim, value_dim, ragged, carried, head_inner=True):
    c = dict(op="decay", mode=mode, n=n, heads=heads, length=length, key_dim=key_dim, value_dim=value_dim, ragged=ragged,
             carried=carried, head_inner=head_inner)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one user's next token on a short cache: nothing but latency
        window_case("window step, one sequence", "forward", 1, 16, 4, 1, 1024, 64, 256, 4, False),
        # a serving batch's next tokens, every sequence at another point of its cache, one slot idle
        window_case("window step, full batch", "forward", 64, 32, 8, 1, 8192, 128, 4096, 4, True),
        # prompts of different lengths in one padded batch, nothing a multiple of anything
        window_case("window prompt, ragged batch", "forward", 4, 16, 4, 1000, 1000, 64, 300, 7, True),
        # a long document: the window is a fraction of it
        window_case("window prompt, long", "forward", 1, 8, 2, 16384, 16384, 128, 2048, 16, False),
        # the next piece of a prompt that is fed piece by piece onto its cache, all of it visible
        window_case("prompt piece on a cache", "forward", 2, 16, 16, 500, 9000, 96, 0, 0, True, False),
        # training at the attention shape of this repository's benchmark (4 x 16 heads, 1024 tokens, 64 per head)
        window_case("window training, short", "train", 4, 16, 16, 1024, 1024, 64, 256, 4, False),
        # training on long sequences with shared K/V heads
        window_case("window training, long", "train", 1, 32, 8, 8192, 8192, 128, 1024, 4, False),
        # one user's next token: latency
        decay_case("decay step, one sequence", "forward", 1, 16, 1, 64, 64, False, True),
        # a serving batch's next tokens: the states are read and written, nothing else counts
        decay_case("decay step, full batch", "forward", 256, 32, 1, 128, 128, False, True),
        # prompts of different lengths in one padded batch
        decay_case("decay prompt, ragged batch", "forward", 4, 16, 1000, 64, 64, True, False),
        # a long document, few heads: the sequence has to be worked on in parallel
        decay_case("decay prompt, long", "forward", 1, 16, 32768, 128, 128, False, True),
        # training on segments of longer sequences: the state is carried in, its gradient out
        decay_case("decay training", "train", 4, 16, 4096, 128, 128, False, True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(2.0 ** rng.uniform(math.log2(lo), math.log2(hi))))))


def draw(rng):
    """One more case: sizes spread over the logarithm, odd ones among them, within the largest listed work."""
    limit = [max(work(c)[k] for c in listed()) for k in ("bytes", "flops")]
    while True:
        heads = rng.choice([1, 2, 4, 6, 8, 12, 16, 24, 32])
        inner = rng.random() < 0.75
        mode = "train" if rng.random() < 0.35 else "forward"
        if rng.random() < 0.55:
            kv_heads = rng.choice([k for k in (1, 2, 3, 4, 6, 8, 12, 16, 24, 32) if heads % k == 0])
            dim = rng.choice([32, 64, 64, 80, 96, 112, 128, 128])
            window = rng.choice([0, _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)])
            sinks = rng.choice([0, 1, 4, 16, _log_int(rng, 1, 200)])
            kind = rng.choice(["step", "piece", "prompt", "prompt"]) if mode == "forward" else "prompt"
            kv_len = _log_int(rng, 64, 16384)
            q_len = {"step": 1, "piece": _log_int(rng, 2, kv_len), "prompt": kv_len}[kind]
            c = window_case(None, mode, _log_int(rng, 1, 64), heads, kv_heads, q_len, kv_len, dim, window, sinks,
                            rng.random() < 0.5, inner)
            scores = c["n"] * heads * q_len * kv_len
        else:
            step = mode == "forward" and rng.random() < 0.3
            length = 1 if step else _log_int(rng, 2, 32768)
            dk = rng.choice([32, 64, 64, 96, 128, 128])
            dv = rng.choice([dk, dk, 64, 128])
            c = decay_case(None, mode, _log_int(rng, 1, 256 if step else 16), heads, length, dk, dv,
                           not step and rng.random() < 0.5, step or rng.random() < 0.5, inner)
            scores = c["n"] * heads * length * 128
        w = work(c)
        if w["bytes"] <= limit[0] and w["flops"] <= limit[1] and scores <= 2 ** 31:
            return c


def _lengths(c):
    """Queries and keys of every sequence: full, or spread down from full, with an idle slot where there are four."""
    n = c["n"]
    kv, q = (c["kv_len"], c["q_len"]) if c["op"] == "window" else (c["length"], c["length"])
    if not c["ragged"]:
        return [q] * n, [kv] * n
    if q == 1:
        vl = [max(1, kv * (n - i) // n) for i in range(n)]
        ql = [1] * n
    elif q == kv:
        vl = [max(1, kv * (n - i) // n) for i in range(n)]
        ql = list(vl)
    else:
        ql = [max(1, q * (n - i) // n) for i in range(n)]
        vl = [max(ql[i], kv * (n - i) // n) for i in range(n)]
    if n >= 4:
        ql[-1] = vl[-1] = 0
    return ql, vl


def work(c):
    ql, vl = _lengths(c)
    if c["op"] == "window":
        H, G, d, W, S = c["heads"], c["kv_heads"], c["head_dim"], c["window"], c["sinks"]
        pairs = keys = 0
        for a, b in zip(ql, vl):
            for i in range(a):
                p = i + b - a
                if W == 0 or p < W + S:
                    pairs += p + 1
                else:
                    pairs += W + S
            if a:
                first = 0 if W == 0 else max(0, b - a - W + 1)
                keys += b - first + min(S, first)
        q = sum(ql)
        if c["mode"] == "forward":
            return {"bytes": 4 * d * (2 * H * q + 2 * G * keys), "flops": 4 * d * H * pairs}
        return {"bytes": 4 * d * (4 * H * q + 4 * G * keys), "flops": 14 * d * H * pairs}
    H, dk, dv = c["heads"], c["key_dim"], c["value_dim"]
    t = sum(vl)
    state = c["n"] * H * dk * dv
    if c["mode"] == "forward":
        return {"bytes": 4 * (H * t * 2 * (dk + dv) + state * (1 + c["carried"])), "flops": 4 * H * t * dk * dv}
    return {"bytes": 4 * (H * t * (4 * dk + 3 * dv) + state * (1 + 3 * c["carried"])), "flops": 10 * H * t * dk * dv}


# ---------------------------------------------------------------- inputs

def _shape(c, heads, length, dim):
    return (c["n"], length, heads, dim) if c["head_inner"] else (c["n"], heads, length, dim)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    c = case
    s = {"case": c}
    ql, vl = _lengths(c)
    s["lens"] = (torch.tensor(ql, dtype=torch.int32, device=DEV), torch.tensor(vl, dtype=torch.int32, device=DEV))
    if c["op"] == "window":
        d = c["head_dim"]
        s["q"] = normal(*_shape(c, c["heads"], c["q_len"], d))
        s["k"] = normal(*_shape(c, c["kv_heads"], c["kv_len"], d))
        s["v"] = normal(*_shape(c, c["kv_heads"], c["kv_len"], d))
        s["scale"] = d ** -0.5
        if c["mode"] == "train":
            s["dy"] = normal(*_shape(c, c["heads"], c["q_len"], d))
    else:
        dk, dv, H = c["key_dim"], c["value_dim"], c["heads"]
        s["q"] = normal(*_shape(c, H, c["length"], dk))
        s["k"] = normal(*_shape(c, H, c["length"], dk))
        s["v"] = normal(*_shape(c, H, c["length"], dv))
        s["scale"] = dk ** -0.5
        # heads forget over a few tokens up to a few thousand
        s["g"] = -torch.exp2(-1.0 - 10.0 * (torch.arange(H, device=DEV) + torch.rand(H, generator=g, device=DEV)) / H)
        s["state"] = normal(c["n"], H, dk, dv) * 4 if c["carried"] else None
        if c["mode"] == "train":
            s["dy"] = normal(*_shape(c, H, c["length"], dv))
            s["dstate"] = normal(c["n"], H, dk, dv) if c["carried"] else None
    if own:
        _prepare_own(s)
    return s


# ---------------------------------------------------------------- the library's calls

def _library():
    package = os.path.join(os.getcwd(), "dragon-alpha-v1.2_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import dragon_hip
    return dragon_hip


def _at(t):
    return 0 if t is None else t.data_ptr()


def _prepare_own(s):
    """What a user's program keeps between calls: outputs and the calls' work buffer."""
    dh, c = _library(), s["case"]
    s["dh"] = dh
    s["y"] = torch.empty_like(s["q"]) if c["op"] == "window" else torch.empty_like(s["v"])
    train = c["mode"] == "train"
    if c["op"] == "window":
        A = dh.Cuda_attention
        d = c["head_dim"]
        sizes = (c["n"], c["heads"], c["kv_heads"], c["q_len"], c["kv_len"], d, d)
        need = A.window_bufsize(*sizes, c["window"], c["sinks"])
        if train:
            need = max(need, A.window_backward_bufsize(*sizes, c["window"], c["sinks"]))
            s["lse"] = torch.empty(c["n"], c["heads"], c["q_len"], device=DEV)
        else:
            s["lse"] = None
        s["args"] = sizes + (c["head_inner"], s["scale"], c["window"], c["sinks"])
    else:
        L = dh.Cuda_linear_attention
        sizes = (c["n"], c["heads"], c["length"], c["key_dim"], c["value_dim"])
        need = L.bufsize(*sizes)
        if train:
            need = max(need, L.backward_bufsize(*sizes))
        s["state_out"] = torch.empty(c["n"], c["heads"], c["key_dim"], c["value_dim"], device=DEV)
        s["dstate_in"] = torch.empty_like(s["state_out"]) if train and c["carried"] else None
        s["args"] = sizes + (c["head_inner"], s["scale"])
    s["buf"] = torch.empty(max(need, 16) // 4, device=DEV)
    s["buf_size"] = need
    if train:
        s["grads"] = [torch.empty_like(s[x]) for x in "qkv"]


def _run_own(s):
    dh, c = s["dh"], s["case"]
    stream = [torch.cuda.current_stream().cuda_stream]
    q, k, v, y = _at(s["q"]), _at(s["k"]), _at(s["v"]), _at(s["y"])
    lens = [_at(t) if c["ragged"] else 0 for t in s["lens"]]
    buf, size = _at(s["buf"]), s["buf_size"]
    if c["op"] == "window":
        A = dh.Cuda_attention
        A.window_forward(stream, 1, q, k, v, y, _at(s["lse"]), lens[0], lens[1], buf, size, *s["args"])
        if c["mode"] == "forward":
            return [s["y"]]
        A.window_backward(stream, 1, q, k, v, y, _at(s["lse"]), _at(s["dy"]), *map(_at, s["grads"]), lens[0], lens[1], buf,
                          size, *s["args"])
        return [s["y"]] + s["grads"]
    L = dh.Cuda_linear_attention
    g = _at(s["g"])
    L.forward(stream, 1, q, k, v, g, _at(s["state"]), y, _at(s["state_out"]), lens[1], buf, size, *s["args"])
    out = [s["y"], s["state_out"]]
    if c["mode"] == "forward":
        return out
    L.backward(stream, 1, q, k, v, g, _at(s["state"]), _at(s["dy"]), _at(s["dstate"]), *map(_at, s["grads"]),
               _at(s["dstate_in"]), lens[1], buf, size, *s["args"])
    return out + s["grads"] + ([s["dstate_in"]] if c["carried"] else [])


# ---------------------------------------------------------------- the plain form

def _by_head(c, x):
    return x.transpose(1, 2) if c["head_inner"] else x


def _plain_window(s):
    c = s["case"]
    n, H, KV, QL, VL, d = c["n"], c["heads"], c["kv_heads"], c["q_len"], c["kv_len"], c["head_dim"]
    G = H // KV
    q = _by_head(c, s["q"]).reshape(n, KV, G * QL, d)
    k = _by_head(c, s["k"])
    v = _by_head(c, s["v"])
    ql, vl = (t.long()[:, None, None] for t in s["lens"])
    i = torch.arange(QL, device=DEV)[None, :, None]
    j = torch.arange(VL, device=DEV)[None, None, :]
    pos = i + vl - ql
    sees = (i < ql) & (j < vl) & (j <= pos)
    if c["window"]:
        sees &= (j > pos - c["window"]) | (j < c["sinks"])
    sees = sees[:, None, None]
    p = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(n, KV, G, QL, VL)
    p.masked_fill_(~sees, float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, torch.ones_like(total), total))
    p = p.view(n, KV, G * QL, VL)
    y = torch.matmul(p, v)

    def out(x, heads):
        return _by_head(c, x.reshape(n, heads, -1, d)).contiguous()

    if c["mode"] == "forward":
        return [out(y, H)]
    dy = _by_head(c, s["dy"]).reshape(n, KV, G * QL, d)
    dv = torch.matmul(p.transpose(2, 3), dy)
    ds = torch.matmul(dy, v.transpose(2, 3)).sub_((dy * y).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3), q)
    return [out(y, H), out(dq, H), out(dk, KV), out(dv, KV)]


CHUNK = 128


def _mix(x, y, z, g, ahead):
    """sum over j <= i (ahead: j >= i) of e^(g |i-j|) <x_i, y_j> z_j, chunk by chunk: [n, H, chunks, CHUNK, dim]"""
    n, H, m, C, _ = x.shape
    at = torch.arange(C, device=DEV, dtype=torch.float64)
    g = g.double()[:, None, None]
    if ahead:
        far, seen = at[None, :] - at[:, None], at[None, :] >= at[:, None]
        to, since = C - 1 - at + 1, at
    else:
        far, seen = at[:, None] - at[None, :], at[:, None] >= at[None, :]
        to, since = at + 1, C - 1 - at
    near = torch.where(seen, torch.exp(g * far.clamp(min=0)), torch.zeros_like(far)).float()[None, :, None]
    to = torch.exp(g * to[:, None]).float()[None, :, None]
    since = torch.exp(g * since[:, None]).float()[None, :, None]
    whole = torch.exp(g * C).float()[None]
    out = torch.matmul(torch.matmul(x, y.transpose(3, 4)) * near, z)
    parts = torch.matmul((y * since).transpose(3, 4), z)
    before = torch.zeros_like(parts)
    run = torch.zeros_like(parts[:, :, 0])
    for i in (range(m - 1, -1, -1) if ahead else range(m)):
        before[:, :, i] = run
        run = run * whole + parts[:, :, i]
    return out + torch.matmul(x * to, before)


def _plain_decay_step(s):
    """A single token: the recurrence itself."""
    c = s["case"]
    q, k, v = (_by_head(c, s[x])[:, :, 0] for x in "qkv")
    state = k[..., :, None] * v[..., None, :]
    if c["carried"]:
        state += torch.exp(s["g"])[None, :, None, None] * s["state"]
    y = torch.matmul(q[..., None, :] * s["scale"], state)
    return [_by_head(c, y).contiguous(), state]


def _plain_decay(s):
    c = s["case"]
    n, H, L = c["n"], c["heads"], c["length"]
    if L == 1 and c["mode"] == "forward" and not c["ragged"]:
        return _plain_decay_step(s)
    C = min(CHUNK, L)
    m = (L + C - 1) // C
    i = torch.arange(L, device=DEV)
    vl = s["lens"][1].long()[:, None, None, None]
    live = (i[None, None, :, None] < vl)

    def rows(x):
        return torch.where(live, _by_head(c, x), torch.zeros((), device=DEV))

    def chunks(x):
        return torch.nn.functional.pad(x, (0, 0, 0, m * C - L)).view(n, H, m, C, -1)

    def whole(x):
        return x.reshape(n, H, m * C, -1)[:, :, :L]

    def out(x):
        return _by_head(c, torch.where(live, x, torch.zeros((), device=DEV))).contiguous()

    q, k, v = rows(s["q"]) * s["scale"], rows(s["k"]), rows(s["v"])
    g = s["g"].double()[None, :, None, None]
    since = torch.where(live, torch.exp(g * (vl - 1 - i[None, None, :, None]).clamp(min=0)), torch.zeros_like(g)).float()
    to = torch.exp(g * (i[None, None, :, None] + 1)).float()
    kept = torch.exp(g * vl).float()
    y = whole(_mix(chunks(q), chunks(k), chunks(v), s["g"], False))
    state = torch.matmul((k * since).transpose(2, 3), v)
    if c["carried"]:
        y = y + torch.matmul(q * to, s["state"])
        state = state + kept * s["state"]
    if c["mode"] == "forward":
        return [out(y), state]
    dy = rows(s["dy"]) * s["scale"]
    raw = rows(s["q"])
    dq = whole(_mix(chunks(dy), chunks(v), chunks(k), s["g"], False))
    dk = whole(_mix(chunks(v), chunks(dy), chunks(raw), s["g"], True))
    dv = whole(_mix(chunks(k), chunks(raw), chunks(dy), s["g"], True))
    if not c["carried"]:
        return [out(y), state, out(dq), out(dk), out(dv)]
    dq = dq + torch.matmul(dy * to, s["state"].transpose(2, 3))
    dk = dk + torch.matmul(v * since, s["dstate"].transpose(2, 3))
    dv = dv + torch.matmul(k * since, s["dstate"])
    dstate = torch.matmul((raw * to).transpose(2, 3), dy) + kept * s["dstate"]
    return [out(y), state, out(dq), out(dk), out(dv), dstate]


def run(state):
    if own:
        return _run_own(state)
    return _plain_window(state) if state["case"]["op"] == "window" else _plain_decay(state)


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return _exact_window(s) if case["op"] == "window" else _exact_decay(s)


def _exact_window(s):
    """Sequence by sequence and block of queries by block, over the keys that a block can see."""
    c = s["case"]
    H, KV, d, W, S = c["heads"], c["kv_heads"], c["head_dim"], c["window"], c["sinks"]
    train = c["mode"] == "train"
    G = H // KV
    q, k, v = (_by_head(c, s[x]) for x in "qkv")
    y = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    if train:
        dy = _by_head(c, s["dy"])
        dq, dk, dv = torch.zeros_like(y), *(torch.zeros(k.shape, dtype=torch.float64, device=DEV) for _ in "kv")
    ql, vl = _lengths(c)
    for n in range(c["n"]):
        a, b = ql[n], vl[n]
        for i0 in range(0, a, 256):
            i = torch.arange(i0, min(a, i0 + 256), device=DEV)
            pos = i + (b - a)
            low = 0 if W == 0 else max(0, i0 + b - a - W + 1)
            j = torch.cat([torch.arange(0, min(S, low), device=DEV),
                           torch.arange(low, min(b, int(pos[-1]) + 1), device=DEV)])
            if j.numel() == 0:
                continue
            seen = j[None] <= pos[:, None]
            if W:
                seen &= (pos[:, None] - j[None] < W) | (j[None] < S)
            for h in range(KV):
                hs = slice(h * G, h * G + G)
                qb, kb, vb = q[n, hs, i].double(), k[n, h, j].double(), v[n, h, j].double()
                logit = torch.where(seen, (qb @ kb.T) * s["scale"], torch.full((), -float("inf"), dtype=torch.float64, device=DEV))
                p = torch.softmax(logit, -1)
                p = torch.where(seen.any(-1)[:, None], p, torch.zeros_like(p))
                yb = p @ vb
                y[n, hs, i] = yb
                if train:
                    db = dy[n, hs, i].double()
                    ds = p * (db @ vb.T - (db * yb).sum(-1, keepdim=True)) * s["scale"]
                    dq[n, hs, i] = ds @ kb
                    m = j.numel()
                    dk[n, h, j] += ds.reshape(-1, m).T @ qb.reshape(-1, d)
                    dv[n, h, j] += p.reshape(-1, m).T @ db.reshape(-1, d)
    outs = [y] + ([dq, dk, dv] if train else [])
    return [_by_head(c, x).contiguous() for x in outs]


def _exact_decay(s):
    """The recurrence, token by token; None where that takes too long."""
    c = s["case"]
    n, H, L, dk, dv = c["n"], c["heads"], c["length"], c["key_dim"], c["value_dim"]
    train = c["mode"] == "train"
    if L * (n * H * dk * dv * 8 * 10 / 3e12 + 60e-6) * (3 if train else 1) > 15:
        return None
    q, k, v = (_by_head(c, s[x]).double() for x in "qkv")
    vl = s["lens"][1].long()
    lam = torch.exp(s["g"].double())[None, :, None, None]
    S = s["state"].double().clone() if c["carried"] else torch.zeros(n, H, dk, dv, dtype=torch.float64, device=DEV)
    y = torch.zeros(n, H, L, dv, dtype=torch.float64, device=DEV)
    dq = torch.zeros_like(q)
    if train:
        dy = _by_head(c, s["dy"]).double()
    for t in range(L):
        on = (t < vl)[:, None, None, None]
        S = torch.where(on, lam * S + k[:, :, t, :, None] * v[:, :, t, None, :], S)
        live = on[:, :, 0].double() * s["scale"]
        y[:, :, t] = (q[:, :, t, :, None] * S).sum(2) * live
        if train:
            dq[:, :, t] = (dy[:, :, t, None, :] * S).sum(3) * live
    outs = [y, dq, torch.zeros_like(k), torch.zeros_like(v)] if train else [y]
    state = S
    if train:
        R = s["dstate"].double().clone() if c["carried"] else torch.zeros_like(S)
        for t in range(L - 1, -1, -1):
            on = (t < vl)[:, None, None, None]
            here = R + q[:, :, t, :, None] * dy[:, :, t, None, :] * s["scale"]
            live = on[:, :, 0].double()
            outs[2][:, :, t] = (here * v[:, :, t, None, :]).sum(3) * live
            outs[3][:, :, t] = (here * k[:, :, t, :, None]).sum(2) * live
            R = torch.where(on, lam * here, R)
    outs = [_by_head(c, x).contiguous() for x in outs]
    outs.insert(1, state)
    return outs + ([R] if train and c["carried"] else [])
