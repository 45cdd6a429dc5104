"""The operators of SAE training, as measured: the router of a routed (switch)
SAE, the gradient of the top-k SAE and the AdamW step.

Each operator has a plain form in elementary torch operations and the call a
user makes of this package (``own``).  Both take the same state.

route        experts of each token from its logits, and the logits' gradient
sae_grad     gradients of x_hat = b_dec + sum_j vals_j W_dec[idxs_j] and of
             vals = X . W_enc[idxs] + b_enc[idxs] from x_hat's gradient
adamw        one AdamW step over all tensors, states in 32 or 8 bits
"""
import math
import os
import sys

import torch

own = False

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2, "": 0}
E4M3 = torch.float8_e4m3fn
BLOCK = 256             # elements of a tensor that share one scale of an 8-bit state
TINY = 2.0 ** -100      # a block whose largest magnitude is below this is stored as zeros
E4M3_MIN = 2.0 ** -9    # the smallest positive E4M3 value
LR, BETA1, BETA2, EPS, DECAY = 3e-4, 0.9, 0.999, 1e-8, 0.01


def package():
    """This repository's package (asked for by the framework's own calls alone)."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "streamtopk-sae_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import streamtopk_sae
    return streamtopk_sae


def listed():
    route = {"op": "route", "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renorm": True,
             "padded": False, "grad": False}
    sae = {"op": "sae_grad", "bias_std": 0.1, "dx": False, "padded": False}
    adamw = {"op": "adamw", "sets": 1, "copy": "", "packed": False}
    return [
        # one activation routed to one of 32 dictionaries, as an interactive probe asks: latency alone
        dict(route, name="route 1 token of 32", N=1, E=32, k=1, dtype="bf16"),
        # a training batch of a switch SAE: one dictionary a token, weighted by its probability, with the gradient
        dict(route, name="route 4096x128 switch", N=4096, E=128, k=1, dtype="fp32", renorm=False, grad=True),
        # many small experts chosen within groups, with a balance bias, the batch's tail padding
        dict(route, name="route 20000x256 grouped", N=20000, E=256, k=8, dtype="fp32", score="sigmoid", bias=True,
             groups=8, top_groups=4, padded=True),
        # a large harvest of activations, routed and back
        dict(route, name="route 131072x64 top4", N=131072, E=64, k=4, dtype="bf16", grad=True),
        # the smallest encode configuration: B=32, d=768, F=16384, k=32 in fp32
        dict(sae, name="grad 32x768 F16384", B=32, d=768, F=16384, k=32, dtype="fp32"),
        # the 1-GPU encode configuration
        dict(sae, name="grad 128x768 F65536", B=128, d=768, F=65536, k=32, dtype="bf16"),
        # odd sizes, features that fire on very many tokens, padded rows, and X's own gradient (a layer below learns too)
        dict(sae, name="grad 1001x1032 F20000 dx", B=1001, d=1032, F=20000, k=33, dtype="fp16", bias_std=1.0, dx=True,
             padded=True),
        # a training batch of a wide dictionary: every feature fires on several tokens
        dict(sae, name="grad 4096x2048 F65536", B=4096, d=2048, F=65536, k=64, dtype="bf16"),
        # one small SAE with states in 32 bits, as in a sweep of many
        dict(adamw, name="adamw 512x64", F=512, d=64, bits=32, param="fp32", grad="fp32"),
        # the smallest encode configuration's dictionary, states in 32 bits
        dict(adamw, name="adamw 16384x768", F=16384, d=768, bits=32, param="fp32", grad="fp32"),
        # one SAE for each of 24 layers, odd widths, bf16 gradients in one packed buffer, states in 8 bits
        dict(adamw, name="adamw 24 SAEs 8-bit", sets=24, F=2001, d=769, bits=8, param="fp32", grad="bf16",
             packed=True),
        # the training batch's dictionary: fp32 weights, the bf16 copy that the encoder reads, states in 8 bits
        dict(adamw, name="adamw 65536x2048 8-bit", F=65536, d=2048, bits=8, param="fp32", grad="bf16", copy="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("route", "sae_grad", "adamw"))
        if op == "route":
            E = rng.choice((8, 16, 60, 64, 128, 160, 256, 512, rng.randint(2, 600)))
            groups = rng.choice((1, 1, 4, 8)) if E % 8 == 0 else 1
            top = rng.randint(1, groups)
            k = min(_log(rng, 1, 16), top * (E // groups))
            c = {"op": op, "N": _log(rng, 1, 131072), "E": E, "k": k, "score": rng.choice(("softmax", "sigmoid")),
                 "bias": rng.random() < 0.5, "groups": groups, "top_groups": top, "renorm": rng.random() < 0.5,
                 "padded": rng.random() < 0.3, "grad": rng.random() < 0.5, "dtype": rng.choice(("fp32", "fp16", "bf16"))}
        elif op == "sae_grad":
            F = _log(rng, 256, 262144)
            d = rng.choice((64, 512, 768, 1024, 2048, 4096, 8 * rng.randint(8, 500), rng.randint(33, 2000)))
            c = {"op": op, "B": _log(rng, 1, 4096), "d": d, "F": F, "k": min(_log(rng, 1, 128), F),
                 "dtype": rng.choice(("fp32", "fp16", "bf16")), "bias_std": rng.choice((0.1, 0.1, 1.0)),
                 "dx": rng.random() < 0.3, "padded": rng.random() < 0.3}
        else:
            bits = rng.choice((8, 32))
            param = rng.choice(("fp32", "fp32", "bf16"))
            c = {"op": op, "sets": _log(rng, 1, 32), "F": _log(rng, 64, 65536), "d": _log(rng, 16, 2048), "bits": bits,
                 "param": param, "grad": rng.choice(("fp32", "bf16")) if param == "fp32" else "bf16",
                 "copy": rng.choice(("", "bf16", "fp16")) if param == "fp32" else "", "packed": rng.random() < 0.5}
        if _cost(c) <= most and (op != "sae_grad" or c["B"] * c["k"] * c["d"] <= 4096 * 64 * 2048):
            return c


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def work(c):
    if c["op"] == "route":
        N, E, k, es = c["N"], c["E"], c["k"], BYTES[c["dtype"]]
        size = N * E * es + N * k * 8 + (E * 4 if c["bias"] else 0) + (N if c["padded"] else 0) + E * 4
        flops = N * E * 4
        if c["grad"]:
            size += N * k * 4 + N * E * es
            flops += N * k * 8
        return {"bytes": size, "flops": flops}
    if c["op"] == "sae_grad":
        B, d, F, k, es = c["B"], c["d"], c["F"], c["k"], BYTES[c["dtype"]]
        used = F * -math.expm1(B * math.log1p(-min(k / F, 1 - 1e-12)))  # dictionary rows that the batch reads
        size = B * d * (4 + es) + used * d * es + 2 * F * d * es + F * 4 + d * 4 + B * k * 12
        flops = 6 * B * k * d
        if c["dx"]:
            size += used * d * es + B * d * es
            flops += 2 * B * k * d
        return {"bytes": size, "flops": flops}
    n = sum(_sizes(c))
    state = 2 * 4 if c["bits"] == 32 else 2 * (1 + 4 / BLOCK)
    return {"bytes": n * (2 * BYTES[c["param"]] + BYTES[c["grad"]] + 2 * state + BYTES[c["copy"]]), "flops": 14 * n}


def _sizes(c):
    """Elements of each tensor of an AdamW case: W_enc, b_enc, W_dec, b_dec of each SAE."""
    return [c["F"] * c["d"], c["F"], c["F"] * c["d"], c["d"]] * c["sets"]


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"route": _prepare_route, "sae_grad": _prepare_sae, "adamw": _prepare_adamw}[case["op"]](case, gen)


def _randn(gen, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)


def _prepare_route(c, gen):
    N, E, k = c["N"], c["E"], c["k"]
    logits = _randn(gen, N, E, std=1.5, dtype=DT[c["dtype"]])
    s = {"case": c, "logits": logits, "bias": _randn(gen, E, std=0.05) if c["bias"] else None, "mask": None,
         "grad_weights": _randn(gen, N, k) if c["grad"] else None}
    if c["padded"]:  # the batch's tail is padding, and holds what memory held
        s["mask"] = torch.arange(N, device="cuda") < max(1, N - N // 10)
        logits[~s["mask"]] = float("nan")
    return s


def _prepare_sae(c, gen):
    B, d, F, k, dt = c["B"], c["d"], c["F"], c["k"], DT[c["dtype"]]
    X = _randn(gen, B, d, dtype=dt)
    W_enc = _randn(gen, F, d, std=d ** -0.5, dtype=dt)
    W_dec = _randn(gen, F, d, std=d ** -0.5, dtype=dt)
    scores = (X @ W_enc.T).float() + _randn(gen, F, std=c["bias_std"])
    vals, idxs = torch.topk(scores, k, dim=1)
    del scores
    idxs = idxs.to(torch.int32)
    if c["padded"]:  # rows behind the last one of a batch carry no codes
        idxs[B - B // 8:] = -1
    # the gradient of the reconstruction error, summed over features and averaged over the batch
    g = _randn(gen, B, d, std=2.0 / B ** 0.5)
    return {"case": c, "g": g, "X": X, "W_enc": W_enc, "W_dec": W_dec, "vals": vals.contiguous(), "idxs": idxs}


def _flat(c, dtype):
    """One buffer for all tensors and each one's view: each at a multiple of 64 elements, or one behind the other."""
    at, views = 0, []
    for n in _sizes(c):
        views.append((at, n))
        at += n if c["packed"] else -(-n // 64) * 64
    buf = torch.zeros(at, dtype=dtype, device="cuda")
    return buf, [buf[a:a + n] for a, n in views]


def _prepare_adamw(c, gen):
    shapes = [(c["F"], c["d"]), (c["F"],), (c["F"], c["d"]), (c["d"],)] * c["sets"]
    pb, p = _flat(c, DT[c["param"]])
    gb, g = _flat(c, DT[c["grad"]])
    s = {"case": c, "step": 100, "p": p, "g": g, "p_all": pb, "g_all": gb, "copy": None, "copy_all": None}
    pb.copy_(torch.randn(pb.shape, generator=gen, device="cuda").mul_(c["d"] ** -0.5))
    gb.copy_(torch.randn(gb.shape, generator=gen, device="cuda").mul_(1e-3))
    for t, shape in zip(g, shapes):  # features that no token of the batch chose have no gradient
        if len(shape) == 2:
            t.view(shape)[torch.rand(shape[0], generator=gen, device="cuda") < 0.3] = 0
    s["copy_all"], s["copy"] = _flat(c, DT[c["copy"]]) if c["copy"] else (None, None)
    if c["bits"] == 32:
        s["m_all"], s["m"] = _flat(c, torch.float32)
        s["v_all"], s["v"] = _flat(c, torch.float32)
        s["m_all"].copy_(torch.randn(pb.shape, generator=gen, device="cuda").mul_(2e-4))
        s["v_all"].copy_(torch.randn(pb.shape, generator=gen, device="cuda").square_().mul_(1e-7))
        s["ms"] = s["vs"] = None
    else:
        s["m_all"], s["m"] = _flat(c, E4M3)
        s["v_all"], s["v"] = _flat(c, E4M3)
        # codes as an earlier step left them: the largest magnitude of a block near 448
        m = torch.randn(pb.shape, generator=gen, device="cuda").mul_(140).clamp_(-448, 448)
        s["m_all"].copy_(m)
        s["v_all"].copy_(m.normal_(generator=gen).abs_().mul_(140).clamp_(2.0 ** -9, 448))
        del m
        blocks = [-(-n // BLOCK) for n in _sizes(c)]
        for name, unit in (("ms", 5e-7), ("vs", 1e-6)):
            s[name + "_all"] = torch.rand(sum(blocks), generator=gen, device="cuda").add_(0.5).mul_(unit)
            s[name] = list(torch.split(s[name + "_all"], blocks))
    for name in ("p", "g", "m", "v", "copy"):
        if s[name] is not None:
            s[name] = [t.view(shape) for t, shape in zip(s[name], shapes)]
    return s


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(s):
    return {"route": _run_route, "sae_grad": _run_sae, "adamw": _run_adamw}[s["case"]["op"]](s)


def _run_route(s):
    c = s["case"]
    if own:
        stk = package()
        how = {"score": c["score"], "renormalize": c["renorm"], "scale": 2.5}
        weights, experts, counts = stk.route_experts(
            s["logits"], c["k"], bias=s["bias"], n_groups=c["groups"], topk_groups=c["top_groups"],
            row_mask=s["mask"], return_counts=True, **how)
        out = {"weights": weights, "experts": experts, "counts": counts}
        if c["grad"]:
            out["logits"] = stk.route_experts_backward(s["grad_weights"], s["logits"], experts, **how)
        return out
    out = _plain_route(s["logits"], s["bias"], s["mask"], c)
    if c["grad"]:
        out["logits"] = _plain_route_grad(s["grad_weights"], s["logits"], out["experts"], c)
    return out


def _scores(logits, c):
    """Each expert's score in 64 bits (chosen experts must not depend on rounding), 0 where the logit is -inf or NaN."""
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    if c["score"] == "sigmoid":
        return x, 1 / (1 + torch.exp(-x))
    top = x.amax(1, keepdim=True)
    e = torch.where(x == -math.inf, 0.0, torch.where(x == top, 1.0, torch.exp(x - top)))
    return x, e / e.sum(1, keepdim=True).clamp_min(1e-300)


def _plain_route(logits, bias, mask, c):
    N, E, k, G = c["N"], c["E"], c["k"], c["groups"]
    x, scores = _scores(logits, c)
    # without a bias experts rank by logit, as both scores rise with it
    choice = x if bias is None else torch.where(x == -math.inf, -math.inf, scores + bias.double())
    if G > 1:  # the groups with the largest sums of their two best
        each = (scores if bias is None else choice).view(N, G, E // G)
        best = each.masked_fill(choice.view(N, G, E // G) == -math.inf, -math.inf).sort(dim=2, descending=True).values[:, :, :2]
        total = torch.where(best == -math.inf, 0.0, best).sum(2).masked_fill(best[:, :, 0] == -math.inf, -math.inf)
        kept = total.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros(N, G, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        choice = choice.masked_fill(~keep.repeat_interleave(E // G, 1), -math.inf)
    best, experts = choice.sort(dim=1, descending=True, stable=True)
    best, experts = best[:, :k], experts[:, :k]
    live = best > -math.inf
    if mask is not None:
        live &= mask[:, None]
    w = torch.where(live, scores.gather(1, experts), 0.0)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300 if c["score"] == "softmax" else 1e-20)
    experts = torch.where(live, experts, -1)
    counts = torch.zeros(E + 1, dtype=torch.int32, device=x.device)
    counts.index_add_(0, (experts.reshape(-1) + E + 1) % (E + 1), torch.ones(N * k, dtype=torch.int32, device=x.device))
    return {"weights": (2.5 * w).float(), "experts": experts.int(), "counts": counts[:E]}


def _plain_route_grad(gw, logits, experts, c):
    x, scores = _scores(logits, c)
    live = experts >= 0
    at = experts.clamp_min(0).long()
    s = torch.where(live, scores.gather(1, at), 0.0)
    g = torch.where(live, 2.5 * gw.double(), 0.0)
    if c["renorm"]:
        low = 1e-300 if c["score"] == "softmax" else 1e-20
        S = s.sum(1, keepdim=True)
        g = torch.where(S >= low, g - (g * s).sum(1, keepdim=True) / S.clamp_min(low), g) / S.clamp_min(low)
    picked = torch.zeros_like(scores).scatter_add_(1, at, g)
    if c["score"] == "sigmoid":
        out = picked * scores * (1 - scores)
    elif c["renorm"]:  # over the chosen alone the sum of g * s is zero
        out = picked * scores
    else:
        out = scores * (picked - (picked * scores).sum(1, keepdim=True))
    return torch.where(live.any(1, keepdim=True), out, 0.0).to(logits.dtype)


def _run_sae(s):
    c, g, X, W_enc, W_dec, vals, idxs = (s[n] for n in ("case", "g", "X", "W_enc", "W_dec", "vals", "idxs"))
    if own:
        r = package().topk_sae_backward(g, X, W_enc, W_dec, vals, idxs, need_dx=c["dx"])
        return {"W_enc": r.W_enc, "b_enc": r.b_enc, "W_dec": r.W_dec, "b_dec": r.b_dec, "vals": r.vals, "X": r.X}
    F, d = W_dec.shape
    B, k = idxs.shape
    live = idxs >= 0
    at = idxs.clamp_min(0).long()
    flat = at.reshape(-1)
    x = X.float()
    dv = torch.where(live, (W_dec[at].float() * g[:, None, :]).sum(2), 0.0)
    v = torch.where(live, vals, 0.0)
    dW_dec = torch.zeros(F, d, device=g.device).index_add_(0, flat, (v[:, :, None] * g[:, None, :]).view(-1, d))
    dW_enc = torch.zeros(F, d, device=g.device).index_add_(0, flat, (dv[:, :, None] * x[:, None, :]).view(-1, d))
    db_enc = torch.zeros(F, device=g.device).index_add_(0, flat, dv.view(-1))
    dX = (dv[:, :, None] * W_enc[at].float()).sum(1).to(X.dtype) if c["dx"] else None
    return {"W_enc": dW_enc.to(W_enc.dtype), "b_enc": db_enc, "W_dec": dW_dec.to(W_dec.dtype), "b_dec": g.sum(0),
            "vals": dv, "X": dX}


def _run_adamw(s):
    s["step"] += 1
    if own:
        package().adamw_step(s["p"], s["g"], s["m"], s["v"], step=s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS,
                             weight_decay=DECAY, exp_avg_scales=s["ms"], exp_avg_sq_scales=s["vs"], copies=s["copy"])
    else:
        for i in range(len(s["p"])):
            _plain_adamw(s, i)
    return [s[n] for n in ("p_all", "m_all", "v_all", "ms_all", "vs_all", "copy_all") if s.get(n) is not None]


def _blocks(t):
    """`t` as rows of BLOCK elements, the last one filled up with zeros."""
    t = t.reshape(-1)
    return torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)).view(-1, BLOCK)


def _encode(t, least):
    """(codes, scales) of an 8-bit state: E4M3 of each block over a 448th of its largest finite magnitude. Where `least`,
    what is not zero is not stored as zero."""
    rows = _blocks(t)
    fine = rows.isfinite()
    top = torch.where(fine, rows, 0.0).abs().amax(1, keepdim=True)
    full = torch.full_like(top, 448.0)
    some = top >= TINY
    q = (rows * (full / torch.where(some, top, 1.0))).clamp(-448, 448).to(E4M3).float()
    if least:
        q = torch.where((rows > 0) & (q == 0), E4M3_MIN, q)
    q = torch.where(some, q, 0.0)
    q = torch.where(fine, q, math.nan).reshape(-1)[: t.numel()].view(t.shape)
    return q.to(E4M3), torch.where(some, top / full, 1.0).view(-1)


def _plain_adamw(s, i):
    step, bits = s["step"], s["case"]["bits"]
    p, g = s["p"][i], s["g"][i].float()
    if bits == 32:
        m, v = s["m"][i], s["v"][i]
    else:
        m, r = ((_blocks(s[q][i].float()) * s[n][i][:, None]).reshape(-1)[: p.numel()].view(p.shape)
                for q, n in (("m", "ms"), ("v", "vs")))
        v = r * r
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + (g * g) * (1 - BETA2)
    root = torch.sqrt(v)
    size = m / (root * (1 / math.sqrt(1 - BETA2 ** step)) + EPS)
    new = p.float() * (1 - LR * DECAY) - size * (LR / (1 - BETA1 ** step))
    p.copy_(new)
    if s["copy"] is not None:
        s["copy"][i].copy_(new)
    if bits == 32:
        s["m"][i].copy_(m)
        s["v"][i].copy_(v)
    else:
        for t, q, n in ((m, "m", "ms"), (root, "v", "vs")):
            codes, scales = _encode(t, q == "v")
            s[q][i].copy_(codes)
            s[n][i].copy_(scales)


# --------------------------------------------------------------------------
# the operators' definition in 64 bits, written apart from the plain forms
# --------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "sae_grad": _exact_sae, "adamw": _exact_adamw}[case["op"]](s)


def _exact_route(s):
    c = s["case"]
    N, E, k, G = c["N"], c["E"], c["k"], c["groups"]
    x = s["logits"].double().nan_to_num(-math.inf, math.inf, -math.inf)
    p = torch.special.expit(x) if c["score"] == "sigmoid" else torch.softmax(x, 1)
    p = p.nan_to_num(0.0)  # rows of padding
    choice = x.clone() if s["bias"] is None else p + s["bias"].double()
    if G > 1:
        per = E // G
        of = (p if s["bias"] is None else choice).view(N, G, per)
        total = of.topk(min(2, per), dim=2).values.sum(2)
        for _ in range(G - c["top_groups"]):  # strike the worst groups, of equals the last
            low = G - 1 - total.flip(1).argmin(1)
            choice.view(N, G, per)[torch.arange(N, device=x.device), low] = -math.inf
            total[torch.arange(N, device=x.device), low] = math.inf
    picks = []
    for _ in range(k):  # the best, of equals the first, and strike it
        picks.append(choice.argmax(1))
        choice[torch.arange(N, device=x.device), picks[-1]] = -math.inf
    experts = torch.stack(picks, 1)
    if s["mask"] is not None:
        experts[~s["mask"]] = -1
    chosen = torch.where(experts >= 0, p.gather(1, experts.clamp_min(0)), 0.0).requires_grad_()
    w = 2.5 * (chosen / chosen.sum(1, keepdim=True).clamp_min(1e-20) if c["renorm"] else chosen)
    out = {"weights": w.detach(), "experts": experts, "counts": None}
    if c["grad"]:  # by differentiation of the scores
        leaf = x.clone().requires_grad_()
        q = torch.special.expit(leaf) if c["score"] == "sigmoid" else torch.softmax(leaf, 1)
        q = q.gather(1, experts.clamp_min(0))
        q = q / q.sum(1, keepdim=True) if c["renorm"] else q
        (2.5 * q * s["grad_weights"].double())[experts[:, 0] >= 0].sum().backward()
        out["logits"] = leaf.grad.nan_to_num(0.0)
    return out


def _exact_sae(s):
    """From the dense codes, as products of whole matrices."""
    c, F = s["case"], s["W_dec"].shape[0]
    B, k = s["idxs"].shape
    g, X = s["g"].double(), s["X"].double()
    at = torch.where(s["idxs"] >= 0, s["idxs"], F).long()
    codes = torch.zeros(B, F + 1, dtype=torch.float64, device=g.device).scatter_(1, at, s["vals"].double())
    dW_dec = codes[:, :F].T @ g
    dense = torch.zeros(B, F + 1, dtype=torch.float64, device=g.device)
    torch.mm(g, s["W_dec"].double().T, out=dense[:, :F])
    dv = dense.gather(1, at)
    del dense
    codes.zero_().scatter_(1, at, dv)
    codes[:, F] = 0
    return {"W_enc": codes[:, :F].T @ X, "b_enc": codes[:, :F].sum(0), "W_dec": dW_dec, "b_dec": g.sum(0), "vals": dv,
            "X": codes[:, :F] @ s["W_enc"].double() if c["dx"] else None}


def _exact_adamw(s):
    c, t = s["case"], s["step"] + 1
    eight = c["bits"] == 8
    outs = {n: s[n].double() for n in ("p_all", "m_all", "v_all", "ms_all", "vs_all", "copy_all") if s.get(n) is not None}
    at = block = 0
    for n in _sizes(c):
        here, nb = slice(at, at + n), -(-n // BLOCK)
        rows = torch.arange(n, device="cuda") // BLOCK
        g = s["g_all"][here].double()
        m, v = s["m_all"][here].double(), s["v_all"][here].double()
        if eight:
            m = m * s["ms_all"][block:block + nb].double()[rows]
            v = (v * s["vs_all"][block:block + nb].double()[rows]) ** 2
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g ** 2
        hat_m, hat_v = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
        p = s["p_all"][here].double()
        p = p - LR * DECAY * p - LR * hat_m / (hat_v.sqrt() + EPS)
        outs["p_all"][here] = p
        if c["copy"]:
            outs["copy_all"][here] = p
        if eight:
            for q, codes, scales in ((m, "m_all", "ms_all"), (v.sqrt(), "v_all", "vs_all")):
                top = torch.zeros(nb, dtype=torch.float64, device="cuda").scatter_reduce_(0, rows, q.abs(), "amax")
                outs[scales][block:block + nb] = top / 448
                code = (q * (448 / top)[rows]).float().to(E4M3).double()
                outs[codes][here] = torch.where((q > 0) & (code == 0) & (codes == "v_all"), E4M3_MIN, code)
        else:
            outs["m_all"][here], outs["v_all"][here] = m, v
        at += n if c["packed"] else -(-n // 64) * 64
        block += nb
    return [outs[n] for n in ("p_all", "m_all", "v_all", "ms_all", "vs_all", "copy_all") if n in outs]

