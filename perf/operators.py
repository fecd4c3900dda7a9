"""What is measured of the plaintext operators around an encrypted prefill.

Three operators run in the clear beside the encrypted graph: rotary positions
(the plain twin of a decoder layer), the matrix-vector product of the client's
head with 4-bit weights (the next token), and the softmax cross entropy over
the vocabulary with its gradient (the score of a prompt, the training of the
head).  ``run`` computes them from elementary torch operations, or with
``own`` through ``easyfhe.plain``.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32,
          "fp64": torch.float64}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "fp64": 8}

VOCAB = 128256  # Llama-3's vocabulary; its decoder layer: 4096, 14336, 32 + 8 heads of 128
IGNORED = -100


def _plain():
    path = os.path.join(os.getcwd(), "easyfhe-llama3-8b_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from easyfhe import plain

    return plain


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def _rope(batch, seq, q_heads, k_heads, dim, rotary, dtype, layout="half", scaling="none",
          grad=False, first=0, fused=False):
    return {"op": "rope", "batch": batch, "seq": seq, "q_heads": q_heads, "k_heads": k_heads,
            "dim": dim, "rotary": rotary, "dtype": dtype, "layout": layout,
            "scaling": scaling, "grad": grad, "first": first, "fused": fused}


def _q4(rows, n, k, group, dtype, zeros=False, scale="bf16", out="same"):
    return {"op": "q4", "rows": rows, "n": n, "k": k, "group": group, "dtype": dtype,
            "zeros": zeros, "scale": scale, "out": out}


def _loss(tokens, vocab, dim, dtype, grads="", ignored=0.0):
    """grads: any of "h" (hidden) and "w" (weight); none: the loss alone."""

    return {"op": "loss", "tokens": tokens, "vocab": vocab, "dim": dim, "dtype": dtype,
            "grads": grads, "ignored": ignored}


def listed():
    named = {
        # one token's queries and keys, far into a long context: latency
        "rope_one_token": _rope(1, 1, 32, 8, 128, 128, "bf16", scaling="bands", first=100003),
        # the plain twin of a layer as the decrypted layer is checked: 128 tokens in binary64
        "rope_layer_fp64": _rope(1, 128, 32, 8, 128, 128, "fp64"),
        # the gradient of an odd batch, interleaved pairs on part of the head, views of a
        # fused q/k/v buffer
        "rope_partial_grad": _rope(3, 1111, 20, 5, 96, 64, "fp16", layout="interleaved",
                                   scaling="yarn", grad=True, first=7, fused=True),
        # a long prompt
        "rope_long": _rope(1, 32768, 32, 8, 128, 128, "bf16", scaling="linear"),
        # a projection of the layer, one token: latency
        "q4_square": _q4(1, 4096, 4096, 128, "bf16"),
        # odd sizes, a last group that is cut short, binary32 rows
        "q4_ragged": _q4(3, 1001, 1000, 32, "fp32", zeros=True, scale="fp16"),
        # the down projection for a few sequences at once, zero points
        "q4_down_rows": _q4(8, 4096, 14336, 64, "fp16", zeros=True, scale="fp16"),
        # the client's next token: one decrypted row (binary32) against the whole head
        "q4_head": _q4(1, VOCAB, 4096, 128, "fp32", out="fp32"),
        # a short prompt's score and its sensitivity, odd sizes, masked tokens
        "loss_small": _loss(45, 32003, 1000, "fp16", grads="h", ignored=0.3),
        # the score of a decrypted prompt of 128 tokens
        "loss_score": _loss(128, VOCAB, 4096, "bf16"),
        # one training step of the head on that prompt
        "loss_step": _loss(128, VOCAB, 4096, "bf16", grads="hw", ignored=0.1),
        # the same on 32 prompts' tokens at once
        "loss_step_large": _loss(4096, VOCAB, 4096, "bf16", grads="hw", ignored=0.1),
    }
    return [{"name": name, **case} for name, case in named.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "q4", "loss"])
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        rotary = dim if rng.random() < 0.6 else 2 * rng.randint(8, dim // 2)
        k_heads = rng.randint(1, 8)
        q_heads = k_heads * rng.randint(1, 4)
        dtype = rng.choice(["bf16", "fp16", "fp32", "fp64"])
        most = 32768 * 40 * 128 * 2 // ((q_heads + k_heads) * dim * SIZE[dtype])
        tokens = _log_int(rng, 1, min(32768, most))
        batch = rng.randint(1, min(4, tokens))
        return _rope(batch, tokens // batch, q_heads, k_heads, dim, rotary, dtype,
                     layout=rng.choice(["half", "interleaved"]),
                     scaling=rng.choice(["none", "linear", "bands", "yarn"]),
                     grad=rng.random() < 0.4, first=_log_int(rng, 1, 1000000),
                     fused=rng.random() < 0.4)
    if op == "q4":
        k = _log_int(rng, 64, 14336)
        n = _log_int(rng, 64, min(VOCAB, VOCAB * 4096 // k))
        return _q4(_log_int(rng, 1, 16), n, k, rng.choice([32, 64, 128]),
                   rng.choice(["bf16", "fp16", "fp32"]), zeros=rng.random() < 0.5,
                   scale=rng.choice(["bf16", "fp16"]), out=rng.choice(["same", "fp32"]))
    return _loss(_log_int(rng, 1, 4096), _log_int(rng, 500, VOCAB),
                 8 * _log_int(rng, 8, 512), rng.choice(["bf16", "fp16"]),
                 grads=rng.choice(["", "h", "w", "hw"]), ignored=rng.choice([0.0, 0.1, 0.5]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

_THETA = 500000.0
_SCALINGS = {
    "none": None,
    "linear": {"type": "linear", "factor": 4.0},
    "bands": {"type": "bands", "factor": 8.0, "low": 1.0, "high": 4.0, "original": 8192},
    "yarn": {"type": "yarn", "factor": 16.0, "original": 4096, "fast": 32.0, "slow": 1.0},
}


def _frequencies(case):
    """Rotations per position (radians) of each pair, and the factor on cos and sin."""

    r = case["rotary"]
    sc = _SCALINGS[case["scaling"]]
    freqs, factor = [], 1.0
    if sc is not None and sc["type"] == "yarn":
        def edge(turns):
            return r * math.log(sc["original"] / (turns * 2 * math.pi)) / (2 * math.log(_THETA))

        low = max(math.floor(edge(sc["fast"])), 0)
        high = min(math.ceil(edge(sc["slow"])), r - 1)
        factor = 0.1 * math.log(sc["factor"]) + 1.0
    for i in range(r // 2):
        f = _THETA ** (-2.0 * i / r)
        if sc is None:
            pass
        elif sc["type"] == "linear":
            f = f / sc["factor"]
        elif sc["type"] == "bands":
            turns = sc["original"] * f / (2 * math.pi)  # within the original context
            if turns < sc["low"]:
                f = f / sc["factor"]
            elif turns <= sc["high"]:
                mix = (turns - sc["low"]) / (sc["high"] - sc["low"])
                f = (1 - mix) * f / sc["factor"] + mix * f
        else:
            ramp = min(max((i - low) / max(high - low, 0.001), 0.0), 1.0)
            f = f / sc["factor"] * ramp + f * (1 - ramp)
        freqs.append(f)
    return freqs, factor


def _heads(case, gen):
    """q, k [batch, seq, heads, dim]: separate, or views of one q/k/v buffer."""

    b, s, d = case["batch"], case["seq"], case["dim"]
    hq, hk = case["q_heads"], case["k_heads"]
    dt = DTYPES[case["dtype"]]
    shape = (b, s, hq + 2 * hk if case["fused"] else hq + hk, d)
    draw_as = torch.float64 if case["dtype"] == "fp64" else torch.float32
    if case["fused"]:
        buf = torch.randn(shape, generator=gen, device="cuda", dtype=draw_as).to(dt)
        return buf[:, :, :hq], buf[:, :, hq:hq + hk]
    q = torch.randn((b, s, hq, d), generator=gen, device="cuda", dtype=draw_as).to(dt)
    k = torch.randn((b, s, hk, d), generator=gen, device="cuda", dtype=draw_as).to(dt)
    return q, k


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    st = {"case": case}
    if case["op"] == "rope":
        st["q"], st["k"] = _heads(case, gen)
        pos = torch.arange(case["seq"], device="cuda", dtype=torch.int64) + case["first"]
        if case["batch"] > 1:  # sequences of a batch start at different places
            start = torch.randint(0, 1000, (case["batch"], 1), generator=gen, device="cuda")
            pos = pos[None, :] + start
        else:
            pos = pos[None, :].contiguous()
        st["positions"] = pos
    elif case["op"] == "q4":
        n, k = case["n"], case["k"]
        groups = -(-k // case["group"])
        st["codes"] = torch.randint(0, 16, (n, k), generator=gen, device="cuda",
                                    dtype=torch.uint8)
        spread = torch.rand((n, groups), generator=gen, device="cuda") + 0.5
        st["scales"] = (spread * (0.25 / math.sqrt(k))).to(DTYPES[case["scale"]])
        st["zeros"] = torch.randint(4, 12, (n, groups), generator=gen, device="cuda",
                                    dtype=torch.uint8) if case["zeros"] else None
        # a normalised hidden state with a few large features
        x = torch.randn((case["rows"], k), generator=gen, device="cuda")
        big = torch.randint(0, k, (max(k // 512, 1),), generator=gen, device="cuda")
        x[:, big] *= 20.0
        st["x"] = x.to(DTYPES[case["dtype"]])
    else:
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        dt = DTYPES[case["dtype"]]
        w = torch.empty((v, d), device="cuda", dtype=dt)
        step = max(1, (1 << 27) // d)
        for v0 in range(0, v, step):  # in pieces: the float draws need not be kept
            n = min(step, v - v0)
            w[v0:v0 + n] = torch.randn((n, d), generator=gen, device="cuda") / math.sqrt(d)
        labels = torch.randint(0, v, (t,), generator=gen, device="cuda")
        # a trained head: the hidden state leans towards its label's row by varying amounts,
        # so the label's probability runs from about 1 / v to nearly 1
        lean = 16.0 * torch.rand((t, 1), generator=gen, device="cuda")
        h = torch.randn((t, d), generator=gen, device="cuda") + lean * w[labels].float()
        st["hidden"], st["weight"] = h.to(dt), w
        off = torch.rand((t,), generator=gen, device="cuda") < case["ignored"]
        st["labels"] = torch.where(off, torch.full_like(labels, IGNORED), labels)
        # the upstream gradient of a weighted mean over the counted tokens
        g = 0.5 + torch.rand((t,), generator=gen, device="cuda")
        st["grad"] = g / t
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "rope":
        if own:
            st["plan"] = _plain().RopePlan(case["dim"], rotary_dim=case["rotary"],
                                           theta=_THETA, layout=case["layout"],
                                           scaling=_SCALINGS[case["scaling"]], device="cuda")
        else:
            freqs, st["factor"] = _frequencies(case)
            st["freqs"] = torch.tensor(freqs, dtype=torch.float64, device="cuda")
    elif case["op"] == "q4" and own:
        st["weight"] = _plain().pack_q4(st.pop("codes"), st.pop("scales"), st.pop("zeros"),
                                        group=case["group"])
    return st


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _pairs(x, r, layout):
    if layout == "half":
        return x[..., :r // 2], x[..., r // 2:r]
    return x[..., 0:r:2], x[..., 1:r:2]


def _run_rope(st):
    case = st["case"]
    r = case["rotary"]
    angles = st["positions"].to(torch.float64)[..., None] * st["freqs"]  # binary64: far positions
    wide = torch.float64 if case["dtype"] == "fp64" else torch.float32
    cos = (torch.cos(angles) * st["factor"]).to(wide)[:, :, None, :]
    sin = (torch.sin(angles) * st["factor"]).to(wide)[:, :, None, :]
    if case["grad"]:
        sin = -sin
    res = {}
    for name in ("q", "k"):
        x = st[name].to(wide)
        x0, x1 = _pairs(x, r, case["layout"])
        y = x.clone()
        y0, y1 = _pairs(y, r, case["layout"])
        y0.copy_(x0 * cos - x1 * sin)
        y1.copy_(x1 * cos + x0 * sin)
        res[name] = y.to(st[name].dtype)
    return res


def _run_q4(st):
    case = st["case"]
    k = case["k"]
    idx = torch.arange(k, device="cuda") // case["group"]
    zero = 8.0 if st["zeros"] is None else st["zeros"].float()[:, idx]
    w = (st["codes"].float() - zero) * st["scales"].float()[:, idx]
    y = st["x"].float() @ w.T
    return y if case["out"] == "fp32" else y.to(st["x"].dtype)


def _run_loss(st):
    case = st["case"]
    h, w, labels = st["hidden"].float(), st["weight"].float(), st["labels"]
    counted = labels != IGNORED
    at = torch.where(counted, labels, torch.zeros_like(labels))[:, None]
    z = h @ w.T
    top = z.max(dim=1, keepdim=True).values
    lse = top + (z - top).exp().sum(dim=1, keepdim=True).log()
    loss = torch.where(counted, (lse - z.gather(1, at))[:, 0], 0.0)
    res = {"loss": loss}
    if case["grads"]:
        dz = z.sub_(lse).exp_()
        dz.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
        dz *= torch.where(counted, st["grad"], 0.0)[:, None]
        if "h" in case["grads"]:
            res["dhidden"] = (dz @ w).to(st["hidden"].dtype)
        if "w" in case["grads"]:
            res["dweight"] = (dz.T @ h).to(st["weight"].dtype)
    return res


def run(state):
    case = state["case"]
    if not own:
        return {"rope": _run_rope, "q4": _run_q4, "loss": _run_loss}[case["op"]](state)
    plain = _plain()
    if case["op"] == "rope":
        f = plain.rope_grad if case["grad"] else plain.rope
        q, k = f(state["q"], state["k"], positions=state["positions"], plan=state["plan"])
        return {"q": q, "k": k}
    if case["op"] == "q4":
        return plain.q4_matvec(state["x"], state["weight"],
                               out_dtype=torch.float32 if case["out"] == "fp32" else None)
    loss, lse = plain.vocab_loss(state["hidden"], state["weight"], state["labels"],
                                 ignore_index=IGNORED)
    res = {"loss": loss}
    if case["grads"]:
        dh, dw = plain.vocab_loss_grad(state["hidden"], state["weight"], state["labels"], lse,
                                       state["grad"], ignore_index=IGNORED,
                                       need_hidden="h" in case["grads"],
                                       need_weight="w" in case["grads"])
        if dh is not None:
            res["dhidden"] = dh
        if dw is not None:
            res["dweight"] = dw
    return res


# ---------------------------------------------------------------------------
# work and definitions
# ---------------------------------------------------------------------------


def work(case):
    if case["op"] == "rope":
        tokens = case["batch"] * case["seq"]
        heads = case["q_heads"] + case["k_heads"]
        return {"bytes": 2 * tokens * heads * case["dim"] * SIZE[case["dtype"]] + 8 * tokens,
                "flops": 3 * tokens * heads * case["rotary"]}
    if case["op"] == "q4":
        n, k, rows = case["n"], case["k"], case["rows"]
        groups = -(-k // case["group"])
        out = 4 if case["out"] == "fp32" else SIZE[case["dtype"]]
        per_group = 2 + (0.5 if case["zeros"] else 0)
        return {"bytes": n * k / 2 + n * groups * per_group + rows * k * SIZE[case["dtype"]]
                + rows * n * out, "flops": 2 * rows * n * k}
    t, v, d = case["tokens"], case["vocab"], case["dim"]
    size = SIZE[case["dtype"]]
    b = (t * d + v * d) * size + t * 8 + t * 4
    products = 1 + len(case["grads"])
    if case["grads"]:
        b += t * 4
    b += t * d * size * ("h" in case["grads"]) + v * d * size * ("w" in case["grads"])
    return {"bytes": b, "flops": 2 * products * t * v * d}


def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "rope":
        r, sign = case["rotary"], -1.0 if case["grad"] else 1.0
        i = torch.arange(r // 2, device="cuda", dtype=torch.float64)
        f, factor = torch.exp(-2.0 * i / r * math.log(_THETA)), 1.0
        if case["scaling"] == "linear":
            f = f / 4.0
        elif case["scaling"] == "bands":  # weight of the unscaled frequency: 0 below 1 turn, 1 above 4
            keep = ((8192 / (2 * math.pi) * f - 1.0) / 3.0).clamp(0.0, 1.0)
            f = f * (keep + (1.0 - keep) / 8.0)
        elif case["scaling"] == "yarn":
            ends = [r / 2 * math.log(4096 / (2 * math.pi * turns)) / math.log(_THETA)
                    for turns in (32.0, 1.0)]
            a, b = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), r - 1)
            keep = 1.0 - ((i - a) / max(b - a, 0.001)).clamp(0.0, 1.0)
            f = f * (keep + (1.0 - keep) / 16.0)
            factor = 1.0 + math.log(16.0) / 10.0
        turn = torch.polar(torch.full_like(f, factor).expand(*st["positions"].shape, -1)
                           .contiguous(), sign * st["positions"][..., None].double() * f)
        res = {}
        for name in ("q", "k"):
            y = st[name].double()
            a = y[..., :r]
            if case["layout"] == "half":
                z = torch.complex(*(p.contiguous() for p in a.chunk(2, dim=-1)))
                z = torch.view_as_real(z * turn[:, :, None])
                y = torch.cat([z[..., 0], z[..., 1], y[..., r:]], dim=-1)
            else:
                z = torch.view_as_complex(a.unflatten(-1, (-1, 2)).contiguous())
                z = torch.view_as_real(z * turn[:, :, None]).flatten(-2)
                y = torch.cat([z, y[..., r:]], dim=-1)
            res[name] = y
        return res
    if case["op"] == "q4":
        x, y = st["x"].double(), []
        for n0 in range(0, case["n"], 8192):
            rows = slice(n0, n0 + 8192)
            acc = 0
            for g in range(st["scales"].shape[1]):
                cols = slice(g * case["group"], min((g + 1) * case["group"], case["k"]))
                c = st["codes"][rows, cols].double()
                c = c - (8 if st["zeros"] is None else st["zeros"][rows, g:g + 1].double())
                acc = acc + (x[:, cols] @ c.T) * st["scales"][rows, g].double()
            y.append(acc)
        return torch.cat(y, dim=1)
    h = st["hidden"].double()
    keep = (st["labels"] != IGNORED).double()
    label = st["labels"].clamp(min=0)
    lse = None
    step = 16384
    pieces = range(0, case["vocab"], step)
    for v0 in pieces:  # log-sum-exp joined over pieces of the vocabulary
        part = torch.logsumexp(h @ st["weight"][v0:v0 + step].double().T, dim=1)
        lse = part if lse is None else torch.logaddexp(lse, part)
    own_logit = (h * st["weight"][label].double()).sum(dim=1)
    res = {"loss": (lse - own_logit) * keep}
    if not case["grads"]:
        return res
    g = st["grad"].double() * keep
    dh = torch.zeros_like(h)
    dw = torch.empty(st["weight"].shape, dtype=torch.float64, device="cuda") \
        if "w" in case["grads"] else None
    for v0 in pieces:
        wp = st["weight"][v0:v0 + step].double()
        p = torch.exp(h @ wp.T - lse[:, None])
        hit = (label[:, None] == torch.arange(v0, v0 + wp.shape[0], device="cuda")[None, :])
        dz = (p - hit.double()) * g[:, None]
        dh += dz @ wp
        if dw is not None:
            dw[v0:v0 + wp.shape[0]] = dz.T @ h
    if "h" in case["grads"]:
        res["dhidden"] = dh
    if dw is not None:
        res["dweight"] = dw
    return res
