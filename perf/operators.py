"""Measured cases of the beam search and distillation operators, with their plain forms.

`own` selects what run() calls: the library's entry points, or the same mathematics in elementary
torch operations.  Shapes follow the library's own workloads (vocabularies of 32000, 32768, 128256,
152064 and 256000 columns, 64 to 1024 rows) and odd sizes next to them.
"""
import math
import os
import sys

import torch

own = False

_HERE = os.path.dirname(os.path.abspath(__file__))
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ESIZE = {"f32": 4, "bf16": 2, "f16": 2}
_INF = float("inf")


def _beam():
    pkg = os.path.join(os.path.dirname(_HERE), "llm-workspace_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import pesti_beam
    return pesti_beam


def _distill():
    _beam()
    import pesti_distill
    return pesti_distill


# ---------------------------------------------------------------- cases

def _select(name, G, W, V, K, dtype, pad=0, masked=False, done=False):
    return {"name": name, "op": "select", "groups": G, "beams": W, "vocab": V, "k": K, "dtype": dtype, "pad": pad,
            "masked": masked, "done": done}


def _advance(name, G, W, K, steps, limit, early):
    return {"name": name, "op": "advance", "groups": G, "beams": W, "k": K, "steps": steps, "limit": limit,
            "early": early}


def _reorder(name, G, W, tensors, heads, room, used, dim, dtype):
    return {"name": name, "op": "reorder", "groups": G, "beams": W, "tensors": tensors, "heads": heads, "room": room,
            "used": used, "dim": dim, "dtype": dtype}


def _dist(name, form, N, V, k, dtype, val, tail, temperature, weighted, pad=0):
    return {"name": name, "op": form, "rows": N, "vocab": V, "k": k, "dtype": dtype, "val": val, "tail": tail,
            "temperature": temperature, "weighted": weighted, "pad": pad}


def listed():
    return [
        # one prompt, four beams: the latency of a decode step's selection
        _select("select_1x4_32000_f32", 1, 4, 32000, 8, "f32"),
        # an odd vocabulary with a grammar's mask and finished groups (rows of every alignment)
        _select("select_13x5_32001_f16_masked", 13, 5, 32001, 10, "f16", masked=True, done=True),
        # a serving batch: 32 prompts of eight beams
        _select("select_32x8_128256_bf16", 32, 8, 128256, 16, "bf16"),
        # offline decoding of many prompts, f32 logits
        _select("select_64x8_152064_f32", 64, 8, 152064, 16, "f32"),
        # the loop control of one prompt's whole search
        _advance("advance_1x4_32", 1, 4, 8, 32, 32, True),
        # of a large batch, up to the length limit
        _advance("advance_128x8_48", 128, 8, 16, 48, 48, False),
        # short caches of one prompt's beams
        _reorder("reorder_1x4_short", 1, 4, 8, 4, 128, 37, 128, "bf16"),
        # the caches of a batch: 2 x 16 tensors with room for 2048 positions, 1100 of them used
        _reorder("reorder_8x8_long", 8, 8, 32, 4, 2048, 1100, 128, "bf16"),
        # loss and its backward pass on a short, odd batch, with the teacher's tail mass
        _dist("loss_33x32001_f32_tail", "loss", 33, 32001, 20, "f32", "f32", True, 2.0, True),
        # a training step's loss and backward pass, teacher renormalised over its list
        _dist("loss_1024x128256_bf16", "loss", 1024, 128256, 64, "bf16", "bf16", False, 1.0, False),
        # loss and gradient in one call: a small step
        _dist("grad_64x32000_f16", "grad", 64, 32000, 32, "f16", "f32", False, 1.5, True, pad=8),
        # and a large one
        _dist("grad_2048x152064_bf16_tail", "grad", 2048, 152064, 64, "bf16", "f32", True, 1.0, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _vocab(rng):
    if rng.random() < 0.4:
        return rng.choice([32000, 32768, 128256, 152064, 256000])
    return _log(rng, 1000, 256000)


def draw(rng):
    op = rng.choice(["select", "select", "select", "advance", "reorder", "loss", "loss", "grad", "grad"])
    if op == "select":
        V = _vocab(rng)
        dtype = rng.choice(["f32", "bf16", "f16"])
        W = _log(rng, 1, 32)
        G = _log(rng, 1, max(1, min(256, 64 * 8 * 152064 // (W * V))))
        K = max(1, min(128, rng.choice([W, 2 * W, 2 * W, 3 * W])))
        return {k: v for k, v in _select("", G, W, V, K, dtype, rng.choice([0, 0, 0, 1, 8]), rng.random() < 0.4,
                                         rng.random() < 0.3).items() if k != "name"}
    if op == "advance":
        W = _log(rng, 1, 16)
        steps = _log(rng, 4, 48)
        return {k: v for k, v in _advance("", _log(rng, 1, 128), W, min(128, 2 * W), steps,
                                          steps + rng.choice([0, 0, 5]), rng.random() < 0.5).items() if k != "name"}
    if op == "reorder":
        W, G = _log(rng, 2, 16), _log(rng, 1, 32)
        room = _log(rng, 16, 2048)
        tensors, heads, dim = rng.randint(1, 32), rng.choice([1, 2, 4, 8]), rng.choice([64, 80, 128])
        while G * W * tensors * heads * room * dim > 64 * 32 * 4 * 2048 * 128:
            G, tensors = max(1, G // 2), max(1, tensors // 2)
        return {k: v for k, v in _reorder("", G, W, tensors, heads, room, rng.randint(1, room), dim,
                                          rng.choice(["bf16", "f16", "f32"])).items() if k != "name"}
    V = _vocab(rng)
    N = _log(rng, 1, min(2048, (2048 * 152064 if op == "grad" else 1024 * 128256) // V))
    dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
    if dtype == "f32":
        N = max(1, N // 2)
    tail = rng.random() < 0.5
    val = "f32" if tail else rng.choice(["f32", "bf16"])
    return {k: v for k, v in _dist("", op, N, V, _log(rng, 1, 256), dtype, val, tail,
                                   rng.choice([1.0, 1.0, 0.7, 2.0, 4.0]), rng.random() < 0.5,
                                   rng.choice([0, 0, 0, 1, 8])).items() if k != "name"}


def work(case):
    c = case
    if c["op"] == "select":
        n = c["groups"] * c["beams"] * c["vocab"]
        return {"bytes": n * _ESIZE[c["dtype"]] + 12 * c["groups"] * c["k"] + 4 * c["groups"] * c["beams"],
                "flops": 4 * n}
    if c["op"] == "advance":
        gw = c["groups"] * c["beams"]
        return {"bytes": 12 * c["steps"] * c["groups"] * c["k"] + 2 * 4 * gw * min(c["steps"], c["limit"]) + 20 * gw,
                "flops": 2 * c["steps"] * c["groups"] * c["k"]}
    if c["op"] == "reorder":
        row = c["heads"] * c["used"] * c["dim"] * _ESIZE[c["dtype"]]
        # about 1 - 1/e of the rows are some beam's parent
        W = c["beams"]
        parents = W * (1.0 - (1.0 - 1.0 / W) ** W)
        return {"bytes": int(c["tensors"] * c["groups"] * (W + parents) * row), "flops": 0}
    n = c["rows"] * c["vocab"]
    return {"bytes": 2 * n * _ESIZE[c["dtype"]] + c["rows"] * c["k"] * (4 + _ESIZE[c["val"]]), "flops": 8 * n}


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * (seed % (1 << 40)) + 17)
    c, s = case, {"case": dict(case)}
    dev = "cuda"

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=dev)

    if c["op"] == "select":
        G, W, V = c["groups"], c["beams"], c["vocab"]
        x = randn(G * W, V + c["pad"]).mul_(3.0)
        if c["masked"]:
            x.masked_fill_(rand(G * W, V + c["pad"]) < 0.3, -_INF)
            x[torch.randint(G * W, (1,), generator=g, device=dev)] = -_INF  # one beam's mask leaves nothing
        s["logits"] = x.to(_DTYPES[c["dtype"]])[:, :V]
        cum = -(rand(G, W) * 3.0).cumsum(1) - 5.0 * rand(G, 1)
        if c["masked"] and W > 2:
            cum[:, -1] = -_INF
        s["cum"] = cum
        s["done"] = (rand(G) < 0.25).to(torch.uint8) if c["done"] else None
    elif c["op"] == "advance":
        G, W, K, T = c["groups"], c["beams"], c["k"], c["steps"]
        step = torch.arange(1, T + 1, device=dev, dtype=torch.float32).view(T, 1, 1)
        s["score"] = -(0.4 * step + (rand(T, G, K) * (3.0 / K)).cumsum(2))
        tok = torch.randint(10, 32000, (T, G, K), generator=g, device=dev)
        tok = torch.where(rand(T, G, K) < 0.05, torch.randint(2, 4, (T, G, K), generator=g, device=dev), tok)
        s["token"] = tok.to(torch.int32)
        s["parent"] = torch.randint(0, W, (T, G, K), generator=g, device=dev).to(torch.int32)
        s["stop"] = [2, 3]
        if own:
            s["state"] = _beam().BeamState(G, W, max_tokens=c["limit"], max_seq_len=4096, stop_tokens=s["stop"],
                                           length_penalty=0.8, early_stop=c["early"])
        else:
            s["stop_t"] = torch.tensor(s["stop"], device=dev)
    elif c["op"] == "reorder":
        n, shape = c["groups"] * c["beams"], (c["groups"] * c["beams"], c["heads"], c["room"], c["dim"])
        dt = _DTYPES[c["dtype"]]
        s["src"] = [randn(*shape).to(dt)[:, :, :c["used"]] for _ in range(c["tensors"])]
        s["dst"] = [torch.zeros(shape, dtype=dt, device=dev)[:, :, :c["used"]] for _ in range(c["tensors"])]
        s["parent"] = torch.randint(0, c["beams"], (c["groups"], c["beams"]), generator=g, device=dev).to(torch.int32)
        assert s["src"][0].shape[0] == n
    else:
        N, V, k, T = c["rows"], c["vocab"], min(c["k"], c["vocab"]), c["temperature"]
        base = randn(N, V).mul_(3.0)
        val, idx = torch.topk(base, k, dim=1)
        s["teacher_lse"] = torch.logsumexp(base / T, 1) if c["tail"] else None
        x = torch.empty(N, V + c["pad"], device=dev, dtype=_DTYPES[c["dtype"]])
        x[:, :V] = base.mul_(0.8).add_(randn(N, V))
        x[:, V:] = 0.0
        del base
        idx = idx.to(torch.int32)
        # some lists are shorter than k (padded as the library's kept lists are)
        short = torch.randint(1, 2 * k + 1, (N, 1), generator=g, device=dev)
        s["idx"] = torch.where(torch.arange(k, device=dev) < short, idx, torch.full_like(idx, -1))
        s["val"] = val.to(_DTYPES[c["val"]])
        s["weight"] = (rand(N) > 0.1).float() * (0.5 + rand(N)) / N if c["weighted"] else None
        s["up"] = 0.5 + rand(N)
        s["logits"] = x[:, :V]
        if own and c["op"] == "loss":
            s["logits"] = s["logits"].detach().requires_grad_()
    return s


# ---------------------------------------------------------------- the plain forms

def _plain_select(s):
    c = s["case"]
    G, W, V, K = c["groups"], c["beams"], c["vocab"], c["k"]
    x = s["logits"]
    x = torch.where(x != x, torch.full_like(x, -_INF), x)
    n = min(K, V)
    order = torch.sort(x, dim=1, descending=True, stable=True)
    top, tok = order.values[:, :n].double(), order.indices[:, :n]
    del order
    m = top[:, :1]
    ref = torch.where(m.isinf(), torch.zeros_like(m), m)
    x = x.double()
    e = torch.where(m == _INF, (x == _INF).double(), torch.exp(x - ref))
    del x
    log_s = torch.log(e.sum(1, keepdim=True))
    del e
    logp = torch.where(m == _INF, torch.where(top == _INF, -log_s, torch.full_like(top, -_INF)), (top - ref) - log_s)
    cum = s["cum"].double().reshape(G * W, 1)
    ok = (top > -_INF) & (logp > -_INF) & (cum > -_INF)
    if s["done"] is not None:
        ok = ok & (s["done"].repeat_interleave(W)[:, None] == 0)
    score = torch.where(ok, cum + logp, torch.full_like(logp, -_INF)).reshape(G, W * n)
    parent = torch.arange(W, device=x_device(s)).repeat_interleave(n).expand(G, W * n)
    if W * n < K:
        more = K - W * n
        score = torch.cat([score, torch.full((G, more), -_INF, device=score.device, dtype=score.dtype)], 1)
        parent = torch.cat([parent, torch.full((G, more), -1, device=score.device)], 1)
        tok = torch.cat([tok.reshape(G, W * n), torch.full((G, more), -1, device=score.device)], 1)
    tok = tok.reshape(G, -1)
    best = torch.sort(score, dim=1, descending=True, stable=True)
    score, at = best.values[:, :K], best.indices[:, :K]
    none = score == -_INF
    minus = torch.full_like(at, -1)
    return (score.float(), torch.where(none, minus, tok.gather(1, at)).int(),
            torch.where(none, minus, parent.gather(1, at)).int())


def x_device(s):
    return s["logits"].device


def _plain_advance(s):
    c = s["case"]
    G, W, K, T, cap = c["groups"], c["beams"], c["k"], c["steps"], min(c["limit"], 4096)
    dev, alpha = s["score"].device, 0.8
    gi, wi = torch.arange(G, device=dev), torch.arange(W, device=dev)
    i64 = dict(device=dev, dtype=torch.int64)
    tokens, fin_tokens = torch.zeros(G, W, cap, **i64), torch.zeros(G, W, cap, **i64)
    count, done, fin_count = torch.zeros(G, **i64), torch.zeros(G, **i64), torch.zeros(G, **i64)
    fin_len, fin_score = torch.zeros(G, W, **i64), torch.full((G, W), -_INF, device=dev)
    cum = torch.full((G, W), -_INF, device=dev)
    cum[:, 0] = 0.0
    last, parent = torch.zeros(G, W, **i64), torch.full((G, W), -1, **i64)

    def insert(when, norm, rows, length):
        nonlocal fin_count
        full = fin_count >= W
        low = fin_score.amin(1, keepdim=True)
        worst = torch.where(fin_score == low, wi, torch.full_like(wi, -1)).amax(1)
        slot = torch.where(full, worst, fin_count.clamp(max=W - 1))
        put = when & (~full | (norm > fin_score[gi, slot]))
        fin_score[gi, slot] = torch.where(put, norm, fin_score[gi, slot])
        fin_len[gi, slot] = torch.where(put, length, fin_len[gi, slot])
        fin_tokens[gi, slot] = torch.where(put[:, None], rows, fin_tokens[gi, slot])
        fin_count = fin_count + (put & ~full).long()

    for t in range(T):
        score, token, par = s["score"][t], s["token"][t].long(), s["parent"][t].long()
        run = (done == 0) & (count < cap)
        done = torch.where((done == 0) & (count >= cap), torch.full_like(done, 2), done)
        live = torch.zeros_like(count)
        n_cum, n_par, n_last = torch.full_like(cum, -_INF), torch.full_like(parent, -1), last.clone()
        by_len = torch.pow((count + 1).double(), alpha)
        for r in range(K):
            sc, tk, pa = score[:, r], token[:, r], par[:, r]
            ok = run & (tk >= 0) & (pa >= 0) & (pa < W)
            stop = ok & (tk[:, None] == s["stop_t"][None]).any(1)
            if r < W:
                insert(stop, (sc.double() / by_len).float(), tokens[gi, pa.clamp(0, W - 1)], count)
            take = ok & ~stop & (live < W)
            slot = live.clamp(max=W - 1)
            n_cum[gi, slot] = torch.where(take, sc, n_cum[gi, slot])
            n_par[gi, slot] = torch.where(take, pa, n_par[gi, slot])
            n_last[gi, slot] = torch.where(take, tk, n_last[gi, slot])
            live = live + take.long()
        moved = n_par >= 0
        rows = tokens[gi[:, None], n_par.clamp(min=0)]
        at = count[:, None, None].expand(G, W, 1).clamp(max=cap - 1)
        rows = rows.scatter(2, at, n_last[:, :, None])
        tokens = torch.where(moved[:, :, None], rows, tokens)
        cum = torch.where(run[:, None], n_cum, cum)
        last = torch.where(run[:, None], n_last, last)
        parent = n_par
        count = count + run.long()
        limit = run & (count >= cap)
        at_limit = torch.pow(count.double(), alpha)
        for w in range(W):
            insert(limit & moved[:, w], (cum[:, w].double() / at_limit).float(), tokens[:, w], count)
        best = cum.amax(1).double()
        ahead = torch.maximum(best / torch.pow((count + 1).double(), alpha), best / float(cap) ** alpha)
        enough = (fin_count >= W) & (c["early"] | (fin_score.amin(1).double() >= ahead))
        code = torch.where(limit, 2, torch.where(run & ((live == 0) | enough), 1, 0))
        done = torch.where(run, code, done)
    return {"tokens": tokens.int(), "count": count.int(), "cum": cum, "last": last.int(), "parent": parent.int(),
            "done": done.to(torch.uint8), "fin_tokens": fin_tokens.int(), "fin_len": fin_len.int(),
            "fin_score": fin_score, "fin_count": fin_count.int()}


def _plain_reorder(s):
    G, W = s["parent"].shape
    p = s["parent"].long()
    itself = torch.arange(W, device=p.device).expand(G, W)
    p = torch.where((p >= 0) & (p < W), p, itself) + torch.arange(G, device=p.device)[:, None] * W
    for a, b in zip(s["src"], s["dst"]):
        b.copy_(a[p.reshape(-1)])
    return s["dst"]


def _plain_distill(s, up):
    """Loss of each row, and the gradient of sum(up * loss) for the logits.

    The loss is a difference of logarithms that nearly cancel once the student is close to its teacher, so what
    is one value for a row or an entry of its list is held in 64 bits; the exponentials of a row are not."""
    T = s["case"]["temperature"]
    x, dt = s["logits"], s["logits"].dtype
    N, V = x.shape
    w = s["weight"] if s["weight"] is not None else torch.ones(N, device=x.device)
    idx = s["idx"].long()
    listed_ = (idx >= 0) & (idx < V)
    at = torch.where(listed_, idx, torch.zeros_like(idx))
    t = s["val"].double() / T
    t = torch.where(listed_, t, torch.full_like(t, -_INF))
    m = x.amax(1, keepdim=True).float()
    m = torch.where(m == -_INF, torch.zeros_like(m), m)
    e = torch.exp((x.float() - m) / T)
    S = e.sum(1, keepdim=True, dtype=torch.float64)
    logp = (x.gather(1, at).double() - m.double()) / T - torch.log(S)
    S1 = torch.where(S == 0, torch.ones_like(S), S)
    member = torch.zeros(N, V + 1, dtype=torch.bool, device=x.device)
    member.scatter_(1, torch.where(listed_, idx, torch.full_like(idx, V)), True)
    member = member[:, :V]
    if s["teacher_lse"] is not None:
        logq = t - s["teacher_lse"].double()[:, None]
        q = torch.exp(logq)
        rest = 1.0 - q.sum(1, keepdim=True)
        q_t = torch.where(rest < 0, torch.zeros_like(rest), rest)
        p_t = torch.where(member, torch.zeros_like(e), e).sum(1, keepdim=True, dtype=torch.float64) / S1
        q_t = torch.where(p_t == 0, torch.zeros_like(q_t), q_t)
    else:
        mt = t.amax(1, keepdim=True)
        logq = t - torch.where(mt == -_INF, torch.zeros_like(mt), mt)
        Z = torch.exp(logq).sum(1, keepdim=True)
        logq = logq - torch.log(torch.where(Z == 0, torch.ones_like(Z), Z))
        q = torch.exp(logq)
        q_t = p_t = torch.zeros_like(S)
    loss = torch.where(q == 0, torch.zeros_like(q), q * (logq - logp)).sum(1)
    loss = loss + torch.where(q_t == 0, torch.zeros_like(q_t), q_t * (torch.log(q_t) - torch.log(p_t))).squeeze(1)
    loss = torch.where(w == 0, torch.zeros_like(loss), w.double() * (T * T) * loss)
    total = q.sum(1, keepdim=True) + q_t
    ratio = torch.where(q_t == 0, torch.zeros_like(q_t), q_t / p_t)
    grad = torch.where(member, e * (total / S1).float(), e * ((total - ratio) / S1).float())
    grad.scatter_add_(1, at, torch.where(listed_, -q, torch.zeros_like(q)).float())
    scale = (up * w * T)[:, None]
    grad = torch.where(w[:, None] == 0, torch.zeros_like(grad), grad * scale)
    return loss.float(), grad.to(dt)


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "select":
            return _plain_select(s)
        if c["op"] == "advance":
            return _plain_advance(s)
        if c["op"] == "reorder":
            return _plain_reorder(s)
        up = s["up"] if c["op"] == "loss" else torch.ones_like(s["up"])
        return _plain_distill(s, up)
    if c["op"] == "select":
        return _beam().beam_select(s["logits"], c["beams"], c["k"], cum=s["cum"], done=s["done"])
    if c["op"] == "advance":
        st = s["state"]
        st.reset()
        for t in range(c["steps"]):
            st.advance(s["score"][t], s["token"][t], s["parent"][t])
        return {"tokens": st.tokens, "count": st.count, "cum": st.cum, "last": st.last, "parent": st.parent,
                "done": st.done, "fin_tokens": st.fin_tokens, "fin_len": st.fin_len, "fin_score": st.fin_score,
                "fin_count": st.fin_count}
    if c["op"] == "reorder":
        return _beam().beam_reorder(s["src"], s["parent"], out=s["dst"])
    more = dict(temperature=c["temperature"], teacher_lse=s["teacher_lse"], weight=s["weight"])
    if c["op"] == "loss":
        loss = _distill().distill_topk(s["logits"], s["idx"], s["val"], **more)
        grad, = torch.autograd.grad(loss, s["logits"], s["up"])
        return loss.detach(), grad
    return _distill().distill_topk_grad(s["logits"], s["idx"], s["val"], **more)


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_select(s):
    c = s["case"]
    G, W, V, K = c["groups"], c["beams"], c["vocab"], c["k"]
    score = torch.full((G, K), -_INF, dtype=torch.float64)
    token, parent = torch.full((G, K), -1, dtype=torch.int32), torch.full((G, K), -1, dtype=torch.int32)
    logits = s["logits"].reshape(G, W, V)
    for g in range(G):
        if s["done"] is not None and int(s["done"][g]):
            continue
        x = logits[g].double()
        flat = (torch.log_softmax(x, 1) + s["cum"][g].double()[:, None]).reshape(-1)
        flat = torch.where(flat.isnan(), torch.full_like(flat, -_INF), flat)
        least = torch.topk(flat, min(K, W * V)).values[-1]
        at = torch.nonzero((flat >= least) & (flat > -_INF)).squeeze(1)
        have = sorted(zip((-flat[at]).tolist(), at.tolist()))[:K]
        for r, (neg, i) in enumerate(have):
            score[g, r], token[g, r], parent[g, r] = -neg, i % V, i // V
    return score, token, parent


def _exact_advance(s):
    c, alpha = s["case"], 0.8
    G, W, cap = c["groups"], c["beams"], min(c["limit"], 4096)
    score, token, par = (s[k].cpu().tolist() for k in ("score", "token", "parent"))
    out = {k: [] for k in ("tokens", "count", "cum", "last", "parent", "done", "fin_tokens", "fin_len", "fin_score",
                           "fin_count")}
    for g in range(G):
        hist, cum = [[] for _ in range(W)], [0.0] + [-_INF] * (W - 1)
        last, parent, pool, count, done = [0] * W, [-1] * W, [], 0, 0

        def finish(norm, toks):
            if len(pool) < W:
                pool.append((norm, toks))
                return
            i = min(range(W), key=lambda j: (pool[j][0], -j))
            if norm > pool[i][0]:
                pool[i] = (norm, toks)

        for t in range(c["steps"]):
            parent = [-1] * W
            if done:
                continue
            if count >= cap:
                done = 2
                continue
            beams = []
            for r in range(c["k"]):
                sc, tk, pa = score[t][g][r], token[t][g][r], par[t][g][r]
                if tk in s["stop"]:
                    if r < W:
                        finish(sc / (count + 1) ** alpha, list(hist[pa]))
                elif len(beams) < W:
                    beams.append((sc, tk, pa))
            new = [hist[pa] + [tk] for _, tk, pa in beams]
            hist = new + hist[len(new):]
            cum = [b[0] for b in beams] + [-_INF] * (W - len(beams))
            last = [b[1] for b in beams] + last[len(beams):]
            parent = [b[2] for b in beams] + [-1] * (W - len(beams))
            count += 1
            if count >= cap:
                for w in range(len(beams)):
                    finish(cum[w] / count ** alpha, list(hist[w]))
                done = 2
            elif not beams:
                done = 1
            elif len(pool) >= W:
                ahead = max(max(cum) / (count + 1) ** alpha, max(cum) / cap ** alpha)
                if c["early"] or min(p[0] for p in pool) >= ahead:
                    done = 1
        out["tokens"].append([h + [0] * (cap - len(h)) for h in hist])
        out["count"].append(count)
        out["cum"].append(cum)
        out["last"].append(last)
        out["parent"].append(parent)
        out["done"].append(done)
        pool += [(-_INF, [])] * (W - len(pool))
        out["fin_tokens"].append([h + [0] * (cap - len(h)) for _, h in pool])
        out["fin_len"].append([len(h) for _, h in pool])
        out["fin_score"].append([p for p, _ in pool])
        out["fin_count"].append(sum(p > -_INF for p, _ in pool))
    kinds = {"cum": torch.float64, "fin_score": torch.float64, "done": torch.uint8}
    return {k: torch.tensor(v, dtype=kinds.get(k, torch.int32)) for k, v in out.items()}


def _exact_distill(s, up):
    T = s["case"]["temperature"]
    x = s["logits"].detach()
    N, V = x.shape
    rows, losses, grads = max(1, (1 << 26) // V), [], []
    for a in range(0, N, rows):
        b = min(N, a + rows)
        xs = x[a:b].double().requires_grad_()
        logp = torch.log_softmax(xs / T, 1)
        idx = s["idx"][a:b].long()
        has = idx >= 0
        at = idx.clamp(min=0)
        t = s["val"][a:b].double() / T
        if s["teacher_lse"] is None:
            logq = torch.log_softmax(t.masked_fill(~has, -_INF), 1)
        else:
            logq = (t - s["teacher_lse"][a:b].double()[:, None]).masked_fill(~has, -_INF)
        q = logq.exp()
        kl = (q * (logq - logp.gather(1, at))).masked_fill(~has, 0.0).sum(1)
        if s["teacher_lse"] is not None:
            rest = (1.0 - q.sum(1)).clamp(min=0.0)
            other = torch.ones(b - a, V, dtype=torch.bool, device=x.device)
            i, j = torch.nonzero(has, as_tuple=True)
            other[i, idx[i, j]] = False
            log_rest = torch.logsumexp(logp.masked_fill(~other, -_INF), 1)
            kl = kl + torch.where(rest > 0, rest * (rest.clamp(min=1e-300).log() - log_rest), torch.zeros_like(rest))
        w = s["weight"][a:b].double() if s["weight"] is not None else torch.ones_like(kl)
        loss = w * T * T * kl
        (loss * up[a:b].double()).sum().backward()
        losses.append(loss.detach())
        grads.append(xs.grad)
    return torch.cat(losses), torch.cat(grads)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        return _exact_select(s)
    if case["op"] == "advance":
        return _exact_advance(s)
    if case["op"] == "reorder":
        W = case["beams"]
        p = s["parent"].cpu().tolist()
        rows = [g * W + w for g, line in enumerate(p) for w in line]
        return [a[rows].double() for a in s["src"]]
    up = s["up"] if case["op"] == "loss" else torch.ones_like(s["up"])
    return _exact_distill(s, up)
