"""Measured cases of the vocabulary projection's operators, with their plain forms: cross entropy straight from the
hidden states and the projection's weight (loss, gradients, scoring), the projection's weight in 4 bits with group
scales (quantised and read back), and logits from it.

`own` selects what run() calls: the library's entry points, or the same mathematics in elementary torch operations.
Vocabularies are the library's own workloads' (32000, 32768, 128256, 152064 and 256000 tokens) and odd ones next to
them, hidden sizes 512 to 4096 and odd ones between.
"""
import math
import os
import sys

import torch

own = False

_HERE = os.path.dirname(os.path.abspath(__file__))
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ESIZE = {"f32": 4, "bf16": 2, "f16": 2}


def _head():
    pkg = os.path.join(os.path.dirname(_HERE), "llm-workspace_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import pesti_head
    return pesti_head


# ---------------------------------------------------------------- cases

def _loss(name, form, N, V, D, dtype, padded=0.0, weighted=False, smoothing=0.0, z_loss=0.0):
    return {"name": name, "op": form, "rows": N, "vocab": V, "dim": D, "dtype": dtype, "padded": padded,
            "weighted": weighted, "smoothing": smoothing, "z_loss": z_loss}


def _quant(name, V, D, group, dtype):
    return {"name": name, "op": "quantize", "vocab": V, "dim": D, "group": group, "dtype": dtype}


def _logits(name, B, V, D, group, dtype, out):
    return {"name": name, "op": "logits", "rows": B, "vocab": V, "dim": D, "group": group, "dtype": dtype, "out": out}


def listed():
    return [
        # loss and backward pass of a short, odd batch with padded rows: launches and autograd count
        _loss("loss_37x32001x512_bf16", "loss", 37, 32001, 512, "bf16", padded=0.2),
        # a training step of a fine-tune whose prompts are masked: half of the rows are padding
        _loss("loss_2048x128256x2048_bf16", "loss", 2048, 128256, 2048, "bf16", padded=0.5, z_loss=1e-4),
        # loss and both gradients in one call, f16 with a loss scale in the weights, smoothed labels
        _loss("grad_500x32768x1000_f16", "grad", 500, 32768, 1000, "f16", weighted=True, smoothing=0.1),
        # and a large step
        _loss("grad_4096x128256x4096_bf16", "grad", 4096, 128256, 4096, "bf16", padded=0.03),
        # scoring of given continuations, no gradients
        _loss("score_16x152064x2048_bf16", "score", 16, 152064, 2048, "bf16"),
        _loss("score_1024x256000x2048_bf16", "score", 1024, 256000, 2048, "bf16", padded=0.1),
        # a small weight into 4 bits and back, with hidden sizes that do not end with a group
        _quant("quantize_32001x1000_f32_g32", 32001, 1000, 32, "f32"),
        # a large one
        _quant("quantize_128256x4096_bf16_g64", 128256, 4096, 64, "bf16"),
        # logits of one token: the latency of a decode step
        _logits("logits_1x32000x2048_bf16_g32", 1, 32000, 2048, 32, "bf16", "bf16"),
        _logits("logits_1x128256x4096_bf16_g64", 1, 128256, 4096, 64, "bf16", "f32"),
        # an odd batch in full precision
        _logits("logits_5x32001x1000_f32_g128", 5, 32001, 1000, 128, "f32", "f32"),
        # a serving batch
        _logits("logits_48x128256x4096_f16_g64", 48, 128256, 4096, 64, "f16", "f32"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _vocab(rng):
    if rng.random() < 0.4:
        return rng.choice([32000, 32768, 128256, 152064, 256000])
    return _log(rng, 1000, 256000)


def draw(rng):
    op = rng.choice(["loss", "loss", "grad", "score", "quantize", "logits", "logits", "logits"])
    V = _vocab(rng)
    if op in ("loss", "grad", "score"):
        D = rng.choice([512, 768, 1024, 2048, 4096, 8 * _log(rng, 32, 512)])
        while V * D > 128256 * 4096:
            V //= 2
        N = _log(rng, 1, 4096 if op == "grad" else 2048)
        while N * V * D > 4096 * 128256 * 4096:
            N //= 2
        c = _loss("", op, N, V, D, rng.choice(["bf16", "bf16", "f16"]), rng.choice([0.0, 0.1, 0.6]),
                  rng.random() < 0.4, rng.choice([0.0, 0.0, 0.1]), rng.choice([0.0, 0.0, 1e-4]))
    else:
        D = rng.choice([512, 1024, 2048, 4096, _log(rng, 256, 4096)])
        while V * D > 128256 * 4096:
            V //= 2
        group, dtype = rng.choice([32, 64, 128]), rng.choice(["bf16", "f16", "f32"])
        if op == "quantize":
            c = _quant("", V, D, group, dtype)
        else:
            c = _logits("", rng.choice([1, 1, 2, 4, _log(rng, 1, 64), _log(rng, 1, 64)]), V, D, group, dtype,
                        rng.choice(["f32", dtype]))
    return {k: v for k, v in c.items() if k != "name"}


def work(case):
    c = case
    VD, e = c["vocab"] * c["dim"], _ESIZE[c["dtype"]]
    if c["op"] == "quantize":  # there and back
        held = VD // 2 + 2 * c["vocab"] * -(-c["dim"] // c["group"])
        return {"bytes": 2 * VD * e + 2 * held, "flops": 4 * VD}
    N = c["rows"]
    if c["op"] == "logits":
        return {"bytes": VD // 2 + 2 * c["vocab"] * -(-c["dim"] // c["group"]) + N * c["dim"] * e
                + N * c["vocab"] * _ESIZE[c["out"]], "flops": 2 * N * VD}
    # padded rows are neither read nor computed
    rows = int(round(N * (1.0 - c["padded"])))
    grads = c["op"] != "score"
    read = VD * e + rows * c["dim"] * e + 12 * N
    return {"bytes": read + (VD * e + N * c["dim"] * e if grads else 0), "flops": (6 if grads else 2) * rows * VD}


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed % (1 << 40)) + 29)
    c, s, dev = case, {"case": dict(case)}, "cuda"
    V, D, dt = c["vocab"], c["dim"], _DTYPES[c["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    if c["op"] in ("loss", "grad", "score"):
        N = c["rows"]
        head = randn(V, D).mul_(1.5 / math.sqrt(D))
        target = torch.randint(0, V, (N,), generator=g, device=dev)
        # hidden states that lean towards their targets, as a trained model's do
        hidden = randn(N, D) + head[target] * (4.0 * rand(N, 1))
        s["head"], s["hidden"] = head.to(dt), hidden.to(dt)
        del head, hidden
        s["target"] = torch.where(rand(N) < c["padded"], torch.full_like(target, -100), target)
        scale = 64.0 if c["dtype"] == "f16" else 1.0
        s["weight"] = scale * (0.5 + rand(N)) if c["weighted"] else None
        s["up"] = scale * (0.5 + rand(N))
        if own and c["op"] == "loss":
            s["hidden"].requires_grad_()
            s["head"].requires_grad_()
        return s
    # a few columns and rows are larger than the rest, as in a trained projection
    head = randn(V, D).mul_(0.02).mul_(torch.where(rand(D) < 0.01, 8.0, 1.0)).mul_(0.5 + rand(V, 1))
    if c["op"] == "quantize":
        s["head"] = head.to(dt)
        return s
    head = head.to(torch.bfloat16)
    s["x"] = randn(c["rows"], D).to(dt)
    if own:
        s["held"] = _head().quantize_head(head, c["group"])
    else:
        s["q"], s["scale"] = _plain_quantize(head, c["group"])
        s["q"] = s["q"].to(torch.int8)
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_cross_entropy(s, up, grads):
    """Loss of each row, and the gradients of sum(up * loss) for the hidden states and the head."""
    c = s["case"]
    h, w, t = s["hidden"].float(), s["head"].float(), s["target"]
    V = w.shape[0]
    live = (t >= 0) & (t < V)
    at = torch.where(live, t, torch.zeros_like(t))[:, None]
    a = torch.where(live, s["weight"] if s["weight"] is not None else torch.ones_like(up), torch.zeros_like(up))
    eps, zeta = c["smoothing"], c["z_loss"]
    z = h @ w.T
    m = z.amax(1, keepdim=True)
    # one value of a row is held in 64 bits: the loss is a difference of near values
    chosen = z.gather(1, at).double()
    mean = z.sum(1, keepdim=True, dtype=torch.float64) / V
    e = torch.exp(z.sub_(m))
    del z
    total = e.sum(1, keepdim=True, dtype=torch.float64)
    lse = m.double() + torch.log(total)
    loss = lse - (1.0 - eps) * chosen - eps * mean + zeta * lse * lse
    loss = torch.where(live, a.double() * loss.squeeze(1), torch.zeros_like(a, dtype=torch.float64)).float()
    if not grads:
        return loss
    g = e.mul_(((1.0 + 2.0 * zeta * lse) / total).float()).sub_(eps / V)
    g.scatter_add_(1, at, torch.full_like(at, -(1.0 - eps), dtype=torch.float32))
    g.mul_((a * up)[:, None])
    g = torch.where(live[:, None], g, torch.zeros_like(g))
    return loss, (g @ w).to(s["hidden"].dtype), (g.T @ h).to(s["head"].dtype)


def _plain_groups(head, group):
    V, D = head.shape
    n = -(-D // group)
    w = torch.zeros(V, n * group, device=head.device, dtype=torch.float32)
    w[:, :D] = head
    return w.view(V, n, group)


def _plain_quantize(head, group):
    """Whole numbers -8 to 7 and each group's scale: a minus eighth of its largest value by magnitude (the first of
    equal ones), rounded to bfloat16."""
    V, D = head.shape
    w = _plain_groups(head, group)
    size = w.abs()
    order = torch.arange(group, device=w.device, dtype=torch.int16)
    first = torch.where(size == size.amax(2, keepdim=True), order, torch.full_like(order, group)).amin(2, keepdim=True)
    del size
    scale = (w.gather(2, first.long()) * -0.125).to(torch.bfloat16)
    # a quotient next to a half needs more than 32 bits
    q = torch.where(scale == 0, torch.zeros((), device=w.device, dtype=torch.float64), torch.round(w.double() / scale.double()))
    return q.clamp_(-8.0, 7.0).float().view(V, -1)[:, :D].contiguous(), scale.squeeze(2)


def _plain_values(q, scale, group):
    return q.float() * scale.float().repeat_interleave(group, 1)[:, :q.shape[1]]


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if own:
        h = _head()
        if op == "quantize":
            held = h.quantize_head(s["head"], c["group"])
            return {"scale": held.scale, "value": held.dequantize(s["head"].dtype)}
        if op == "logits":
            return h.head_logits(s["x"], s["held"], dtype=_DTYPES[c["out"]])
        more = dict(weight=s["weight"], label_smoothing=c["smoothing"], z_loss=c["z_loss"])
        if op == "score":
            return h.linear_cross_entropy(s["hidden"], s["head"], s["target"], **more)
        if op == "grad":
            return h.linear_cross_entropy_grad(s["hidden"], s["head"], s["target"], **more)
        loss = h.linear_cross_entropy(s["hidden"], s["head"], s["target"], **more)
        return (loss.detach(), *torch.autograd.grad(loss, (s["hidden"], s["head"]), s["up"]))
    if op == "quantize":
        q, scale = _plain_quantize(s["head"], c["group"])
        return {"scale": scale, "value": _plain_values(q, scale, c["group"]).to(s["head"].dtype)}
    if op == "logits":
        return (s["x"].float() @ _plain_values(s["q"], s["scale"], c["group"]).T).to(_DTYPES[c["out"]])
    return _plain_cross_entropy(s, s["up"] if op == "loss" else torch.ones_like(s["up"]), op != "score")


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_cross_entropy(s, up, grads):
    c = s["case"]
    w = s["head"].detach().double()
    V = w.shape[0]
    N, D = s["hidden"].shape
    losses, gh, gw = torch.zeros(N, dtype=torch.float64, device=w.device), None, None
    if grads:
        gh, gw = torch.zeros(N, D, dtype=torch.float64, device=w.device), torch.zeros_like(w)
    live = torch.nonzero((s["target"] >= 0) & (s["target"] < V)).squeeze(1)
    per = max(1, (1 << 28) // V)
    for i in live.split(per) if live.numel() else ():
        h, t = s["hidden"].detach()[i].double(), s["target"][i]
        z = h @ w.T
        lse = torch.logsumexp(z, 1)
        a = s["weight"][i].double() if s["weight"] is not None else torch.ones_like(lse)
        nll = lse - z[torch.arange(len(i), device=z.device), t]
        losses[i] = a * ((1.0 - c["smoothing"]) * nll + c["smoothing"] * (lse - z.mean(1)) + c["z_loss"] * lse ** 2)
        if not grads:
            continue
        p = torch.exp_(z - lse[:, None])
        del z
        p *= (1.0 + 2.0 * c["z_loss"] * lse)[:, None]
        p -= c["smoothing"] / V
        p[torch.arange(len(i), device=p.device), t] -= 1.0 - c["smoothing"]
        p *= (a * up[i].double())[:, None]
        gh[i] = p @ w
        gw += p.T @ h
    return (losses, gh, gw) if grads else losses


def _exact_quantize(head, group):
    """(whole numbers, scales) in 64 bits, padded to whole groups."""
    V, D = head.shape
    w = torch.nn.functional.pad(head.double(), (0, -D % group)).view(V, -1, group)
    top, low = w.amax(2), w.amin(2)
    # equal magnitudes of both signs: the sign of the one that comes first
    both = top == -low
    sign_first = torch.where((w == top[:, :, None]).int().argmax(2) < (w == low[:, :, None]).int().argmax(2), top, low)
    most = torch.where(both, sign_first, torch.where(top > -low, top, low))
    scale = (most / -8.0).float().to(torch.bfloat16).double()
    r = w / torch.where(scale == 0, torch.ones_like(scale), scale)[:, :, None]
    q = torch.floor(r)
    up = r - q
    q = q + ((up > 0.5) | ((up == 0.5) & (q % 2 == 1)))
    return torch.where(scale[:, :, None] == 0, torch.zeros_like(q), q.clamp(-8, 7)), scale


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] in ("loss", "grad", "score"):
        return _exact_cross_entropy(s, s["up"] if c["op"] == "loss" else torch.ones_like(s["up"]), c["op"] != "score")
    D, per = c["dim"], max(1, (1 << 27) // c["dim"])
    if c["op"] == "quantize":
        scales, values = [], []
        for a in range(0, c["vocab"], per):
            q, scale = _exact_quantize(s["head"][a:a + per], c["group"])
            scales.append(scale)
            values.append((q * scale[:, :, None]).reshape(q.shape[0], -1)[:, :D].to(
                torch.float32 if c["dtype"] == "f32" else torch.float64))
        return {"scale": torch.cat(scales), "value": torch.cat(values)}
    if "held" in s:
        return None
    x, out = s["x"].double(), []
    for a in range(0, c["vocab"], per):
        w = torch.nn.functional.pad(s["q"][a:a + per].double(), (0, -D % c["group"]))
        w = w.view(w.shape[0], -1, c["group"]) * s["scale"][a:a + per].double()[:, :, None]
        out.append(x @ w.reshape(w.shape[0], -1)[:, :D].T)
    return torch.cat(out, 1)
