"""The operators of a gated, normed feed-forward block of Kronecker-sparse layers and of its training, over the
sizes, types and layouts that a program uses them in: what each computes, in plain torch and by the framework's
kernels, and what it cannot do without.

``kind`` of a case:

``gated``  h = act(G x + bias) * (U x + bias), G and U two factors of one pattern (a, b, c, d) that share x,
           kept side by side: (a*d*c, 2*b), gate columns first
``norm``   r' = r + alpha * gate * P(x), n = norm(r') * weight + bias; P is the norm after the block, with a
           weight of its own, or nothing.  ``groups`` rows of gates: 1 for all rows, or one for each image
``muon``   an update's blocks of c x b made orthogonal by five Newton-Schulz steps; ``step``: momentum before
           and the new weights after it

``train`` returns the results and the gradients of everything; ``bs_last`` is feature-major.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16}
SIZES = {"fp32": 4, "fp16": 2}
FULL = 25088  # 128 images of 196 tokens
NS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-6
NS_EPS = 1e-7
LR, BETA, DECAY = 0.02, 0.95, 0.01


def _gated(name, pattern, dtype, batch, act="silu", bias=True, bs_last=False, train=False):
    case = {"kind": "gated", "pattern": pattern, "dtype": dtype, "batch": batch, "act": act, "bias": bias,
            "bs_last": bs_last, "train": train}
    return dict(case, name=name) if name else case


def _norm(name, features, dtype, batch, norm="rms", post=True, groups=1, bs_last=False, train=False):
    case = {"kind": "norm", "features": features, "dtype": dtype, "batch": batch, "norm": norm, "post": post,
            "groups": groups, "bs_last": bs_last, "train": train}
    return dict(case, name=name) if name else case


def _muon(name, pattern, dtype, parts=1, step=False):
    case = {"kind": "muon", "pattern": pattern, "dtype": dtype, "parts": parts, "step": step}
    return dict(case, name=name) if name else case


def listed():
    return [
        # serving, one token: the gated projection of a 384-wide block
        _gated("gated fp16 one token", "1x768x192x2", "fp16", 1, bias=False),
        # one image of 197 tokens (a class token makes them odd) through blocks of 64 inputs
        _gated("gated fp16 one image", "6x256x64x1", "fp16", 197, act="gelu"),
        # serving full batches
        _gated("gated fp16 full", "1x768x192x2", "fp16", FULL),
        # training in fp32 on dense 192 x 192 blocks, feature-major rows that no vector divides
        _gated("gated fp32 last odd train", "4x192x192x1", "fp32", 33 * 197, act="gelu", bs_last=True, train=True),
        # the training step of the 384-wide block on full batches: the largest
        _gated("gated fp16 train", "1x768x192x2", "fp16", FULL, train=True),
        # serving, one token: both norms around a residual connection
        _norm("norm fp16 one token", 768, "fp16", 1),
        # each image gates the block by its own vector; norm before the next block only
        _norm("norm fp16 gate of image", 768, "fp16", FULL, norm="layer", post=False, groups=128),
        # training with both norms on full batches
        _norm("norm fp16 train", 768, "fp16", FULL, train=True),
        # training in fp32 on feature-major rows that no vector divides
        _norm("norm fp32 last odd train", 384, "fp32", 33 * 197, norm="layer", bs_last=True, train=True),
        # the update of one small factor
        _muon("orthogonal fp32 64x64", "6x64x64x1", "fp32"),
        # the fp16 factor of a 384-wide block's down-projection, with momentum and new weights
        _muon("muon fp16 128x128", "1x128x128x3", "fp16", step=True),
        # the largest pair of projections of a 768-wide block
        _muon("muon fp32 1536x384 pair", "1x1536x384x2", "fp32", parts=2, step=True),
    ]


def _pattern(case):
    return tuple(int(v) for v in case["pattern"].split("x"))


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("gated", "gated", "norm", "norm", "muon"))
    dtype = rng.choice(("fp32", "fp16", "fp16"))
    batch = min(FULL, _log(rng, 1, FULL))
    train = rng.random() < 0.4
    bs_last = rng.random() < 0.4
    if kind == "gated":
        while True:
            c = rng.choice((16, 32, 48, 64, 96, 128, 192, 256, 384))
            b = rng.choice((c, c, 2 * c, 4 * c, max(16, c // 4)))
            if rng.random() < 0.15:
                b += rng.randint(1, 15)
            if rng.random() < 0.15:
                c += rng.randint(1, 15)
            a, d = rng.choice((1, 1, 2, 3, 4, 6, 12, 16)), rng.choice((1, 1, 2, 2, 3, 4, 6, 8, 16))
            if 64 <= a * d * max(b, c) <= 6144:
                break
        case = _gated(None, "%dx%dx%dx%d" % (a, b, c, d), dtype, batch, rng.choice(("silu", "gelu")),
                      rng.random() < 0.5, bs_last, train)
        while _cost(case) > _cost(listed()[4]):
            case["batch"] = (case["batch"] + 1) // 2
    elif kind == "norm":
        features = _log(rng, 32, 8192)
        if rng.random() < 0.7:
            features = max(32, features // 32 * 32)
        groups = 1
        if rng.random() < 0.4:  # whole images
            groups = max(1, batch // 196)
            batch = groups * min(batch, rng.choice((196, 197)))
        case = _norm(None, features, dtype, batch, rng.choice(("rms", "layer")), rng.random() < 0.5, groups,
                     bs_last, train)
        while _cost(case) > _cost(listed()[7]):
            if case["groups"] > 1:
                rows = case["batch"] // case["groups"]
                case["groups"] = (case["groups"] + 1) // 2
                case["batch"] = rows * case["groups"]
            else:
                case["batch"] = (case["batch"] + 1) // 2
    else:
        while True:
            c, b = _log(rng, 4, 512), _log(rng, 4, 768)
            if rng.random() < 0.6:
                b, c = max(16, b // 16 * 16), max(16, c // 16 * 16)
            a, d = rng.choice((1, 1, 2, 4, 6, 12, 16)), rng.choice((1, 1, 2, 3, 4, 16, 64))
            case = _muon(None, "%dx%dx%dx%d" % (a, b, c, d), dtype, rng.choice((1, 2)), rng.random() < 0.5)
            if _cost(case) <= _cost(listed()[11]) and a * b * c * d <= 1 << 20:
                break
    return case


def _cost(case):
    """Seconds of a pass at ordinary rates: what keeps drawn cases below the largest."""
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / (6e13 if case["dtype"] == "fp32" else 3e14)


class _Draws:
    """Values on the GPU from a seed."""

    def __init__(self, seed, dtype):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = dtype

    def normal(self, *shape, scale=1.0, mean=0.0, dtype=None):
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return (t * scale + mean).to(dtype or self.dtype)


def prepare(case, seed):
    """Inputs, parameters and, for training, the gradients of the results."""
    draws, dtype = _Draws(seed, DTYPES[case["dtype"]]), DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["kind"] == "muon":
        a, b, c, d = _pattern(case)
        shape = (a * d * c, case["parts"] * b)
        s["grad"] = draws.normal(*shape, scale=1e-2)
        if case["step"]:
            s["momentum"] = draws.normal(*shape, scale=3e-2, dtype=torch.float32)
            s["weight"] = draws.normal(*shape, scale=1 / math.sqrt(3 * c))
        return s
    batch, bs_last = case["batch"], case["bs_last"]

    def rows(features):
        return draws.normal(*((features, batch) if bs_last else (batch, features)))

    if case["kind"] == "gated":
        a, b, c, d = _pattern(case)
        s["x"] = rows(a * c * d)
        s["factor"] = draws.normal(a * d * c, 2 * b, scale=1 / math.sqrt(c))
        s["bias"] = draws.normal(2 * a * b * d, scale=0.1) if case["bias"] else None
        s["wanted"] = [s["x"], s["factor"]] + ([s["bias"]] if case["bias"] else [])
        if case["train"]:
            s["grads"] = [rows(a * b * d)]
    else:
        h = case["features"]
        s["x"], s["residual"] = rows(h), rows(h)
        s["gate"] = draws.normal(*((case["groups"], h) if case["groups"] > 1 else (h,)), scale=0.3, mean=0.5)
        s["weight"] = draws.normal(h, scale=0.1, mean=1.0)
        s["bias"] = draws.normal(h, scale=0.1) if case["norm"] == "layer" else None
        s["post"] = draws.normal(h, scale=0.1, mean=1.0) if case["post"] else None
        s["wanted"] = [t for t in (s["x"], s["residual"], s["gate"], s["post"], s["weight"], s["bias"])
                       if t is not None]
        if case["train"]:
            s["grads"] = [rows(h), rows(h)]
    if case["train"]:
        for t in s["wanted"]:
            t.requires_grad_(True)
    return s


def run(state):
    case = state["case"]
    if own:
        return _RUN_OWN[case["kind"]](state, case)
    with torch.no_grad():
        return _RUN_PLAIN[case["kind"]](state, case)


# -- the framework's operators ---------------------------------------------------------------------


def _own_gated(s, case):
    from ksmm_amd import gated_linear

    h = gated_linear(s["x"], s["factor"], _pattern(case), bias=s["bias"], act=case["act"], bs_last=case["bs_last"])
    if not case["train"]:
        return [h]
    return [h.detach()] + list(torch.autograd.grad([h], s["wanted"], s["grads"]))


def _own_norm(s, case):
    from ksmm_amd import residual_norm

    r, n = residual_norm(s["x"], s["residual"], gate=s["gate"], post_weight=s["post"], weight=s["weight"],
                         bias=s["bias"], alpha=0.7, norm=case["norm"], eps=EPS, bs_last=case["bs_last"])
    if not case["train"]:
        return [r, n]
    return [r.detach(), n.detach()] + list(torch.autograd.grad([r, n], s["wanted"], s["grads"]))


def _own_muon(s, case):
    from ksmm_amd import muon_update, orthogonalize

    if not case["step"]:
        return [orthogonalize(s["grad"], _pattern(case), parts=case["parts"], steps=STEPS, coefficients=NS,
                              eps=NS_EPS)]
    return list(muon_update(s["weight"], s["grad"], s["momentum"], _pattern(case), parts=case["parts"], lr=LR,
                            beta=BETA, weight_decay=DECAY, nesterov=True, steps=STEPS, coefficients=NS, eps=NS_EPS))


_RUN_OWN = {"gated": _own_gated, "norm": _own_norm, "muon": _own_muon}


# -- in elementary operations, in 32 bits, rounded once ---------------------------------------------


def _act(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))


def _act_slope(name, z):
    if name == "silu":
        g = torch.sigmoid(z)
        return g * (1 + z * (1 - g))
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _plain_gated(s, case):
    a, b, c, d = _pattern(case)
    n, last, dtype = case["batch"], case["bs_last"], DTYPES[case["dtype"]]

    def blocks(t, k):
        """(a, d, n, k): what each block reads or writes."""
        t = t.float()
        return (t.view(a, k, d, n).permute(0, 2, 3, 1) if last else t.view(n, a, k, d).permute(1, 3, 0, 2)).contiguous()

    def tensor(t):
        """Blocks (a, d, n, k) in the layout of the tensors, in their type."""
        k = t.shape[3]
        t = t.permute(0, 3, 1, 2).reshape(a * k * d, n) if last else t.permute(2, 0, 3, 1).reshape(n, a * k * d)
        return t.to(dtype)

    x, w = blocks(s["x"], c), s["factor"].float().view(a, d, c, 2 * b)
    z = torch.matmul(x, w)
    if case["bias"]:
        z = z + s["bias"].float().view(a, 2 * b, d).permute(0, 2, 1).unsqueeze(2)
    g, u = z[..., :b], z[..., b:]
    act = _act(case["act"], g)
    out = [tensor(act * u)]
    if not case["train"]:
        return out
    dh = blocks(s["grads"][0], b)
    dz = torch.cat([dh * u * _act_slope(case["act"], g), dh * act], dim=3)
    out.append(tensor(torch.matmul(dz, w.transpose(2, 3).contiguous())))
    out.append(torch.matmul(x.transpose(2, 3).contiguous(), dz).reshape(a * d * c, 2 * b).to(dtype))
    if case["bias"]:
        out.append(dz.sum(2).permute(0, 2, 1).reshape(-1).to(dtype))
    return out


def _plain_norm(s, case):
    last, dtype = case["bs_last"], DTYPES[case["dtype"]]
    h, groups = case["features"], case["groups"]

    def rows(t):
        return t.float().t() if last else t.float()

    def tensor(t):
        return (t.t().contiguous() if last else t).to(dtype)

    def normed(t):
        if case["norm"] == "layer":
            t = t - t.mean(1, keepdim=True)
        scale = torch.rsqrt(t.square().mean(1, keepdim=True) + EPS)
        return t * scale, scale

    def through(dv, v, scale):
        """The gradient of what was normed to v."""
        dv = dv - v * (dv * v).mean(1, keepdim=True) - (dv.mean(1, keepdim=True) if case["norm"] == "layer" else 0)
        return dv * scale

    def over_group(t):
        return t.view(groups, -1, h)

    x, gate, w = rows(s["x"]), s["gate"].float().view(groups, 1, h), s["weight"].float()
    p = x
    if case["post"]:
        post = s["post"].float()
        u, x_scale = normed(x)
        p = u * post
    r = rows(s["residual"]) + 0.7 * (over_group(p) * gate).view(-1, h)
    v, r_scale = normed(r)
    n = v * w
    if s["bias"] is not None:
        n = n + s["bias"].float()
    out = [tensor(r), tensor(n)]
    if not case["train"]:
        return out
    dr, dn = (rows(g) for g in s["grads"])
    dr = dr + through(dn * w, v, r_scale)
    dgate = 0.7 * (over_group(dr) * over_group(p)).sum(1)
    dx = 0.7 * (over_group(dr) * gate).view(-1, h)
    more = []
    if case["post"]:
        more = [(dx * u).sum(0).to(dtype)]
        dx = through(dx * post, u, x_scale)
    more.append((dn * v).sum(0).to(dtype))
    if s["bias"] is not None:
        more.append(dn.sum(0).to(dtype))
    return out + [tensor(dx), tensor(dr), dgate.view(s["gate"].shape).to(dtype)] + more


def _plain_muon(s, case):
    a, b, c, d = _pattern(case)
    parts, u = case["parts"], s["grad"].float()
    if case["step"]:
        m = BETA * s["momentum"] + u
        u = u + BETA * m
    x = u.view(a * d, c, parts, b).transpose(1, 2).contiguous()
    x = x / (x.square().sum((2, 3), keepdim=True).sqrt() + NS_EPS)
    if c > b:
        x = x.transpose(2, 3).contiguous()
    x = _newton_schulz(x, STEPS)
    if c > b:
        x = x.transpose(2, 3)
    x = x.transpose(1, 2).reshape(a * d * c, parts * b)
    if not case["step"]:
        return [x.to(DTYPES[case["dtype"]])]
    w = (1 - LR * DECAY) * s["weight"].float() - LR * math.sqrt(max(1.0, b / c)) * x
    return [w.to(DTYPES[case["dtype"]]), m]


def _newton_schulz(x, steps):
    if steps == 0:
        return x
    g = torch.matmul(x, x.transpose(2, 3).contiguous())
    return _newton_schulz(NS[0] * x + torch.matmul(NS[1] * g + NS[2] * torch.matmul(g, g), x), steps - 1)


_RUN_PLAIN = {"gated": _plain_gated, "norm": _plain_norm, "muon": _plain_muon}


# -- from the definitions, in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        s = {k: v.detach().double() if torch.is_tensor(v) else v for k, v in s.items()}
        return {"gated": _exact_gated, "norm": _exact_norm, "muon": _exact_muon}[case["kind"]](s, case)


def _exact_gated(s, case):
    """Block by block: its rows and columns of the two sparse matrices."""
    a, b, c, d = _pattern(case)
    x = s["x"].t() if case["bs_last"] else s["x"]
    n = x.shape[0]
    h, dx, dfactor = x.new_empty(n, a * b * d), torch.empty_like(x), torch.empty_like(s["factor"])
    dbias = x.new_zeros(2 * a * b * d)
    dh = None
    if case["train"]:
        dh = s["grads"][0].detach().double()
        dh = dh.t() if case["bs_last"] else dh
    silu = case["act"] == "silu"
    for i in range(a):
        for l in range(d):
            cols = torch.arange(c, device=x.device) * d + i * c * d + l
            outs = torch.arange(b, device=x.device) * d + i * b * d + l
            first = torch.arange(b, device=x.device) * d + 2 * i * b * d + l
            at = (i * d + l) * c
            w, xi = s["factor"][at:at + c], x[:, cols]
            g, u = xi @ w[:, :b], xi @ w[:, b:]
            if case["bias"]:
                g, u = g + s["bias"][first], u + s["bias"][first + b * d]
            phi = torch.reciprocal(1 + torch.exp(-g)) if silu else torch.special.ndtr(g)
            h[:, outs] = g * phi * u
            if dh is None:
                continue
            slope = phi + g * (phi * (1 - phi) if silu else torch.exp(-g * g / 2) / math.sqrt(2 * math.pi))
            du = dh[:, outs] * g * phi
            dg = dh[:, outs] * u * slope
            dx[:, cols] = dg @ w[:, :b].t() + du @ w[:, b:].t()
            dfactor[at:at + c, :b], dfactor[at:at + c, b:] = xi.t() @ dg, xi.t() @ du
            dbias[first], dbias[first + b * d] = dg.sum(0), du.sum(0)
    if case["bs_last"]:
        h, dx = h.t(), dx.t()
    return [h] + ([dx, dfactor] + ([dbias] if case["bias"] else []) if case["train"] else [])


def _exact_norm(s, case):
    axis = 0 if case["bs_last"] else 1
    h, groups, batch = case["features"], case["groups"], case["batch"]

    def along(v):
        """A vector of features, or one for each group, against the tensors."""
        v = v.reshape(-1, h).repeat_interleave(batch // (v.numel() // h), 0)
        return v.t() if axis == 0 else v

    def stats(t):
        mean = t.mean(axis, keepdim=True) if case["norm"] == "layer" else 0.0
        return mean, ((t - mean) ** 2).mean(axis, keepdim=True).add(EPS) ** -0.5

    def to_input(dv, v, rho):
        inner = dv - v * (dv * v).mean(axis, keepdim=True)
        return rho * (inner - dv.mean(axis, keepdim=True)) if case["norm"] == "layer" else rho * inner

    x, gate = s["x"], along(s["gate"])
    p = x
    if case["post"]:
        mean_x, rho_x = stats(x)
        u = (x - mean_x) * rho_x
        p = u * along(s["post"])
    r = s["residual"] + 0.7 * gate * p
    mean_r, rho_r = stats(r)
    v = (r - mean_r) * rho_r
    n = v * along(s["weight"])
    if s["bias"] is not None:
        n = n + along(s["bias"])
    out = [r, n]
    if not case["train"]:
        return out
    dr, dn = (g.detach().double() for g in s["grads"])
    dr = dr + to_input(dn * along(s["weight"]), v, rho_r)
    dp = 0.7 * gate * dr
    more = [(dn * v).sum(1 - axis)]
    if case["post"]:
        more = [(dp * u).sum(1 - axis)] + more
        dx = to_input(dp * along(s["post"]), u, rho_x)
    else:
        dx = dp
    if s["bias"] is not None:
        more.append(dn.sum(1 - axis))
    dgate = 0.7 * dr * p
    dgate = (dgate.t() if axis == 0 else dgate).reshape(groups, -1, h).sum(1).reshape(s["gate"].shape)
    return out + [dx, dr, dgate] + more


def _exact_muon(s, case):
    """A step is an odd polynomial of the singular values."""
    a, b, c, d = _pattern(case)
    u = s["grad"]
    if case["step"]:
        m = u + BETA * s["momentum"]
        u = u + BETA * m
    x = u.cpu().reshape(a * d, c, case["parts"], b).permute(0, 2, 1, 3)
    left, sigma, right = torch.linalg.svd(x, full_matrices=False)
    sigma = sigma / (torch.linalg.vector_norm(sigma, dim=-1, keepdim=True) + NS_EPS)
    for _ in range(STEPS):
        sigma = NS[0] * sigma + NS[1] * sigma ** 3 + NS[2] * sigma ** 5
    x = ((left * sigma.unsqueeze(-2)) @ right).permute(0, 2, 1, 3).reshape(u.shape).to(u.device)
    if not case["step"]:
        return [x]
    return [s["weight"] * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, b / c)) * x, m]


def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "muon":
        a, b, c, d = _pattern(case)
        m, n, blocks = min(b, c), max(b, c), a * d * case["parts"]
        values = blocks * b * c
        # the Gram matrix and its square are symmetric: half of each product is enough
        flops = STEPS * blocks * (m * m * n + m ** 3 + 2 * m * m * n)
        return {"bytes": values * (3 * size + 8 if case["step"] else 2 * size), "flops": flops + 6 * values}
    times = 2 if case["train"] else 1
    if case["kind"] == "gated":
        a, b, c, d = _pattern(case)
        params = 2 * a * b * c * d + (2 * a * b * d if case["bias"] else 0)
        values = case["batch"] * a * d * (b + c)
        return {"bytes": times * size * (params + values),
                "flops": (3 if case["train"] else 1) * 4 * case["batch"] * a * b * c * d}
    h = case["features"]
    params = h * (case["groups"] + 1 + int(case["post"]) + int(case["norm"] == "layer"))
    values = case["batch"] * h
    return {"bytes": times * size * (4 * values + params), "flops": (35 if case["train"] else 12) * values}
