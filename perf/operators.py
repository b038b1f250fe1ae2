"""What the MoE layer's operators for routing, 4-bit experts and 8-bit norms are measured on.

Three kinds of cases: ``route`` (scores, selection bias, expert groups, top-k), ``experts`` (the routed experts'
products with 4-bit weights and group scales) and ``norm`` (residual addition, RMSNorm and an e4m3 output with
scales).  ``run`` computes them in elementary torch operations, or with the framework's kernels where ``own`` is set.
"""

import math

import torch

own = False

E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def _route(name, T, E, K, scoring, groups=1, keep=1, group_score="max", bias=True, closed=0, renorm=True,
           scale=1.0, dtype="fp32"):
    return {"name": name, "kind": "route", "T": T, "E": E, "K": K, "scoring": scoring, "groups": groups,
            "keep": keep, "group_score": group_score, "bias": bias, "closed": closed, "renorm": renorm,
            "scale": scale, "dtype": dtype}


def _experts(name, T, E, K, H, I, skew, group=128, act="silu", dtype="bf16"):
    return {"name": name, "kind": "experts", "T": T, "E": E, "K": K, "H": H, "I": I, "skew": skew, "group": group,
            "act": act, "dtype": dtype}


def _norm(name, T, H, group, residual=True, normed=False, bias=False, dtype="bf16"):
    return {"name": name, "kind": "norm", "T": T, "H": H, "group": group, "residual": residual, "normed": normed,
            "bias": bias, "dtype": dtype}


def listed():
    return [
        # a decode step of one sequence: latency alone counts
        _route("route_token", 1, 64, 6, "softmax", groups=8, keep=3),
        # a decode batch of the 60-expert layer, experts balanced by a bias
        _route("route_decode", 61, 60, 4, "sigmoid"),
        # a prompt through a layer of many experts in groups
        _route("route_prompt", 8192, 256, 8, "sigmoid", groups=8, keep=4, group_score="top2", scale=2.5),
        # the 60-expert decode layer with one sequence (matrix-vector products)
        _experts("experts_token", 1, 60, 4, 2048, 1408, "even"),
        # the same layer with its decode batch, a few experts taking most tokens
        _experts("experts_decode", 64, 60, 4, 2048, 1408, "zipf"),
        # eight large experts, an odd handful of sequences, fine-grained scales
        _experts("experts_wide_few", 7, 8, 2, 4096, 14336, "even", group=32),
        # eight large experts, a short prompt in fp16
        _experts("experts_wide_short", 333, 8, 2, 4096, 14336, "even", group=64, dtype="fp16"),
        # the 64-expert layer's prompt
        _experts("experts_prompt", 8192, 64, 6, 2048, 1408, "even"),
        # the eight-expert layer's prompt
        _experts("experts_wide_prompt", 4096, 8, 2, 4096, 14336, "zipf"),
        # between two decoder layers while decoding: one scale for each token
        _norm("norm_decode", 64, 4096, 0),
        # the same for a prompt, the 16-bit row kept for the router beside the 8-bit one
        _norm("norm_prompt", 8192, 2048, 128, normed=True),
        # a wide row in fp16 without a residual, an odd number of tokens
        _norm("norm_wide", 2047, 6144, 0, residual=False, bias=True, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("route", "experts", "experts", "norm"))
    if kind == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        per = max(2, _log(rng, 8, 512) // groups)
        E = min(1024, per * groups)
        E -= E % groups
        keep = rng.randint(1, groups)
        K = rng.randint(1, min(16, keep * (E // groups)))
        T = max(1, min(_log(rng, 1, 16384), 8192 * 256 // E))
        bias = rng.random() < 0.7
        return {"kind": "route", "T": T, "E": E, "K": K, "scoring": rng.choice(("softmax", "sigmoid")),
                "groups": groups, "keep": keep, "group_score": rng.choice(("max", "top2")), "bias": bias,
                "closed": rng.randint(0, E // 4) if bias and rng.random() < 0.3 else 0,
                "renorm": rng.random() < 0.7, "scale": rng.choice((1.0, 2.5)),
                "dtype": rng.choice(("fp32", "fp32", "bf16", "fp16"))}
    if kind == "experts":
        E = rng.choice((4, 8, 16, 60, 64, 128))
        K = rng.randint(1, min(8, E))
        H = 8 * _log(rng, 16, 512)
        I = 8 * _log(rng, 8, max(9, min(1792, 400_000_000 // (E * H * 8))))
        # the plain form multiplies every token with every expert: kept below the largest listed case
        most = int(min(2.9e12 / (6.0 * K * H * I), 1.1e13 / (6.0 * E * H * I), 6e9 / (8.0 * E * (I + H))))
        T = _log(rng, 1, max(1, min(8192, most)))
        return {"kind": "experts", "T": T, "E": E, "K": K, "H": H, "I": I, "skew": rng.choice(("even", "zipf")),
                "group": rng.choice((32, 64, 128)), "act": rng.choice(("silu", "silu", "gelu", "gelu_tanh")),
                "dtype": rng.choice(("bf16", "bf16", "fp16"))}
    group = rng.choice((0, 0, 32, 64, 128))
    step = group or 8
    H = step * max(1, _log(rng, 64, 16384) // step)
    T = max(1, min(_log(rng, 1, 16384), 8192 * 2048 // H))
    return {"kind": "norm", "T": T, "H": H, "group": group, "residual": rng.random() < 0.7,
            "normed": rng.random() < 0.4, "bias": rng.random() < 0.3, "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32"))}


# ----------------------------------------------------------------- inputs
def _probabilities(E, skew):
    p = [(e + 1) ** -1.1 if skew == "zipf" else 1.0 for e in range(E)]
    return [v / sum(p) for v in p]


def _quantised(E, N, Kd, group, dt, gen):
    """Codes [E, N, Kd/2] (two to a byte, the lower index in the low four bits) and scales of seeded N(0, 0.02)
    weights: the scale of a group is its largest magnitude / 7, rounded to five significant bits."""
    dev = gen.device
    ng = -(-Kd // group)
    codes = torch.empty(E, N, Kd // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(E, N, ng, dtype=dt, device=dev)
    for e in range(E):
        w = torch.zeros(N, ng * group, device=dev)
        w[:, :Kd] = torch.randn(N, Kd, generator=gen, device=dev) * 0.02
        w = w.view(N, ng, group)
        m, ex = torch.frexp(w.abs().amax(-1).clamp_min(1e-3) / 7)
        s = torch.ldexp(torch.round(m * 32) / 32, ex)
        q = (torch.round(w / s[..., None]).clamp(-8, 7) + 8).view(N, ng * group)[:, :Kd].to(torch.uint8)
        codes[e] = q[:, 0::2] | (q[:, 1::2] << 4)
        scales[e] = s.to(dt)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev, dt, T = gen.device, DTYPES[case["dtype"]], case["T"]

    def rn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    s = {"case": case}
    if case["kind"] == "route":
        E = case["E"]
        s["logits"] = rn(T, E).to(dt)
        if case["bias"]:
            s["bias"] = rn(E) * 0.05
            if case["closed"]:
                s["bias"][torch.randperm(E, generator=gen, device=dev)[: case["closed"]]] = -math.inf
        return s
    if case["kind"] == "norm":
        H = case["H"]
        s["x"] = rn(T, H)
        s["x"][:, :: 97] *= 8  # a few channels carry much of the energy, as activations do
        s["x"] = s["x"].to(dt)
        s["residual"] = (rn(T, H) * 2).to(dt) if case["residual"] else None
        s["weight"] = 1 + 0.1 * rn(H)
        s["bias"] = 0.1 * rn(H) if case["bias"] else None
        return s
    E, K, H, I, g = (case[k] for k in ("E", "K", "H", "I", "group"))
    s["x"] = rn(T, H).to(dt)
    s["c1"], s["s1"] = _quantised(E, 2 * I, H, g, dt, gen)
    s["c2"], s["s2"] = _quantised(E, H, I, g, dt, gen)
    p = torch.tensor(_probabilities(E, case["skew"]), device=dev)
    p = p[torch.randperm(E, generator=gen, device=dev)]
    race = torch.empty(T, E, device=dev).exponential_(generator=gen) / p  # the K first are K draws without return
    s["ids"] = torch.topk(race, K, largest=False).indices.to(torch.int32)
    s["weights"] = torch.softmax(rn(T, K), -1)
    if own:  # a program lays its experts out once, when it loads them
        from reframework_b200 import kernels
        s["w1"] = kernels.int4_pack(s["c1"], s["s1"], group_size=g, gated=True)
        s["w2"] = kernels.int4_pack(s["c2"], s["s2"], group_size=g)
    return s


# ------------------------------------------------------------- plain forms
def _plain_route(s):
    c = s["case"]
    T, E, G = c["T"], c["E"], c["groups"]
    # 64 bits: which of two close scores is larger decides the ids
    x = s["logits"].double()
    if c["scoring"] == "softmax":
        score = torch.exp(x - x.amax(-1, keepdim=True))
        score = score / score.sum(-1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score + s["bias"].double() if c["bias"] else score
    if G > 1:
        in_group = torch.sort(choice.view(T, G, E // G), dim=-1, descending=True).values
        of_group = in_group[..., 0] if c["group_score"] == "max" else in_group[..., 0] + in_group[..., 1]
        best = torch.sort(of_group, dim=-1, descending=True, stable=True).indices[:, : c["keep"]]
        kept = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, best, True)
        choice = torch.where(kept[..., None].expand(T, G, E // G).reshape(T, E), choice, -math.inf)
    ids = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, : c["K"]]
    w = torch.gather(score, 1, ids)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-20)
    return [(w * c["scale"]).float(), ids.to(torch.int32)]


def _act(kind, g):
    if kind == "silu":
        return g / (1 + torch.exp(-g))
    if kind == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))


def _plain_weights(codes, scales, group):
    E, N, half = codes.shape
    q = torch.stack((codes & 15, codes >> 4), -1).view(E, N, 2 * half).float().sub_(8)
    full = 2 * half // group * group
    q[..., :full].view(E, N, -1, group).mul_(scales[..., : full // group, None].float())
    if full < 2 * half:
        q[..., full:].mul_(scales[..., -1:].float())
    return q


def _plain_experts(s):
    c = s["case"]
    T, E, I = c["T"], c["E"], c["I"]
    x = s["x"].float().expand(E, T, c["H"])
    gu = torch.bmm(x, _plain_weights(s["c1"], s["s1"], c["group"]).transpose(1, 2))
    h = _act(c["act"], gu[..., :I]) * gu[..., I:]
    y = torch.bmm(h, _plain_weights(s["c2"], s["s2"], c["group"]).transpose(1, 2))
    share = torch.zeros(T, E, device=x.device).scatter_add_(1, s["ids"].long(), s["weights"])
    return [y.mul_(share.t()[..., None]).sum(0).to(s["x"].dtype)]


def _plain_norm(s):
    c = s["case"]
    T, H = c["T"], c["H"]
    r = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    z = r.float()
    z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-6) * s["weight"]
    if s["bias"] is not None:
        z = z + s["bias"]
    zg = z.view(T, -1, c["group"] or H)
    top = zg.abs().amax(-1)
    scale = torch.where(top > 0, top / E4M3_MAX, 1.0)
    q = (zg / scale[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(T, H)
    return [q, scale] + ([r] if c["residual"] else []) + ([z.to(s["x"].dtype)] if c["normed"] else [])


def run(state):
    c = state["case"]
    if not own:
        return {"route": _plain_route, "experts": _plain_experts, "norm": _plain_norm}[c["kind"]](state)
    from reframework_b200 import kernels
    if c["kind"] == "route":
        w, ids, _, _, _ = kernels.router_grouped_topk(
            state["logits"], None, c["K"], scoring=c["scoring"], select_bias=state.get("bias"),
            num_groups=c["groups"], topk_groups=c["keep"], group_score=c["group_score"], renormalize=c["renorm"],
            scale=c["scale"])
        return [w, ids]
    if c["kind"] == "experts":
        return [kernels.moe_experts_int4(state["x"], state["w1"], state["w2"], state["weights"], state["ids"],
                                         activation=c["act"])]
    out = kernels.add_rmsnorm_q8(state["x"], state["weight"], residual=state["residual"], bias=state["bias"],
                                 eps=1e-6, group_size=c["group"], want_normed=c["normed"])
    return [out.q, out.scales] + ([out.residual] if c["residual"] else []) + ([out.normed] if c["normed"] else [])


# -------------------------------------------------------------- work, exact
def work(case):
    T, size = case["T"], DTYPES[case["dtype"]].itemsize
    if case["kind"] == "route":
        E, K = case["E"], case["K"]
        return {"bytes": T * E * size + T * K * 8 + (4 * E if case["bias"] else 0), "flops": 8.0 * T * E}
    if case["kind"] == "norm":
        H = case["H"]
        rows = size * (1 + 2 * case["residual"] + case["normed"]) + 1
        scales = T * (H // case["group"] if case["group"] else 1)
        return {"bytes": T * H * rows + 4 * scales + 4 * H * (1 + case["bias"]), "flops": 8.0 * T * H}
    E, K, H, I, g = (case[k] for k in ("E", "K", "H", "I", "group"))
    # experts that some token reaches, on average over the draws of the routing
    reached = sum(1 - (1 - min(1.0, K * p)) ** T for p in _probabilities(E, case["skew"]))
    weights = 3.0 * H * I / 2 + size * (2 * I * -(-H // g) + H * -(-I // g))
    return {"bytes": max(reached, float(min(K, E))) * weights + 2 * T * H * size + 8.0 * T * K,
            "flops": 6.0 * T * K * H * I}


def exact(case, seed):
    s = prepare(case, seed)
    T = case["T"]
    if case["kind"] == "route":
        E, K, G = case["E"], case["K"], case["groups"]
        x = s["logits"].double()
        score = torch.softmax(x, 1) if case["scoring"] == "softmax" else torch.sigmoid(x)
        pick = score.clone()
        if case["bias"]:
            pick += s["bias"].double()
        ids = torch.arange(E, device=x.device).expand(T, E)
        if G > 1:
            m = E // G
            best = torch.topk(pick.view(T, G, m), 2 if case["group_score"] == "top2" else 1).values.sum(-1)
            # a group stays when fewer than `keep` groups come before it
            before = (best[:, None, :] > best[:, :, None]) | ((best[:, None, :] == best[:, :, None])
                                                             & torch.ones(G, G, device=x.device).tril(-1).bool())
            stays = before.sum(-1) < case["keep"]
            pick[~stays.repeat_interleave(m, 1)] = -math.inf
        order = torch.argsort(-pick, dim=1, stable=True)
        ids = torch.gather(ids, 1, order)[:, :K]
        w = torch.gather(score, 1, ids)
        if case["renorm"]:
            w = w / torch.maximum(w.sum(1, keepdim=True), torch.tensor(1e-20, dtype=w.dtype, device=w.device))
        return [w * case["scale"], ids.to(torch.int32)]
    if case["kind"] == "norm":
        H = case["H"]
        r = s["x"].double()
        if case["residual"]:
            r = (r + s["residual"].double()).to(s["x"].dtype).double()  # the row that is stored is the row that is normed
        z = r * torch.rsqrt(r.pow(2).mean(1, keepdim=True) + 1e-6) * s["weight"].double()
        z = z if s["bias"] is None else z + s["bias"].double()
        parts = z.reshape(-1, case["group"] or H)
        scale = parts.abs().max(1, keepdim=True).values / E4M3_MAX
        scale[scale == 0] = 1
        return ([(parts / scale).reshape(T, H), scale.reshape(T, -1)] + ([r] if case["residual"] else [])
                + ([z] if case["normed"] else []))
    E, I, g = case["E"], case["I"], case["group"]

    def weights(codes, scales):
        low, high = codes.bitwise_and(15), codes.bitwise_right_shift(4)
        q = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
        q[:, 0::2], q[:, 1::2] = low, high
        return (q - 8) * scales.double().repeat_interleave(g, 1)[:, : q.shape[1]]

    out = torch.zeros(T, case["H"], dtype=torch.float64, device=s["x"].device)
    for e in range(E):
        t, k = torch.nonzero(s["ids"] == e, as_tuple=True)
        if not t.numel():
            continue
        gu = s["x"][t].double() @ weights(s["c1"][e], s["s1"][e]).T
        a, u = gu[:, :I], gu[:, I:]
        if case["act"] == "silu":
            a = a * torch.sigmoid(a)
        elif case["act"] == "gelu":
            a = a * (0.5 + 0.5 * torch.erf(a / math.sqrt(2)))
        else:
            a = a * 0.5 * (1 + torch.tanh((a + 0.044715 * a.pow(3)) * math.sqrt(2 / math.pi)))
        out.index_add_(0, t, (a * u) @ weights(s["c2"][e], s["s2"][e]).T * s["weights"][t, k].double()[:, None])
    return [out]
