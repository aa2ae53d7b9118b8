"""Kronecker-sparse products in microscaled 4-bit numbers and the AdamW step, over the sizes, types and layouts that a
program uses them in: what each computes, in plain torch and by the framework's kernels, and what it cannot do without.

``kind`` of a case:

``quantize``  x as 4-bit numbers (e2m1), 32 of them along c with a power of two in common, and the values these stand for
``product``   y = act(W x + bias), W in such numbers and x made such numbers in the call; ``gated``: act(G x) * (U x) of
              two factors side by side, (a*d, 2*b, c), gate rows first
``train``     the same of a factor in 16 or 32 bits, which the call quantises too, and the gradients of everything: those
              of what the quantised values are multiplied with, handed through the roundings
``adamw``     one step of AdamW over many tensors, its moments in 32 bits or in 8: blocks of 32 with a power of two in
              common, e4m3 and unsigned e5m3, rounded up or down by a hash of seed, step and place

``bs_last`` is feature-major.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16}
SIZES = {"fp32": 4, "fp16": 2}
FULL = 25088  # 128 images of 196 tokens
LR, BETAS, EPS, DECAY, STEP, SEED, GRAD_SCALE = 1e-3, (0.9, 0.999), 1e-8, 0.01, 25, 7, 1.0 / 1024
LOWEST = -120  # exponent of a block's scale


def _quantize(name, sizes, dtype, batch, bs_last=False):
    case = {"kind": "quantize", "sizes": sizes, "dtype": dtype, "batch": batch, "bs_last": bs_last}
    return dict(case, name=name) if name else case


def _product(name, pattern, dtype, batch, act="none", bias=False, gated=False, bs_last=False, train=False):
    case = {"kind": "train" if train else "product", "pattern": pattern, "dtype": dtype, "batch": batch, "act": act,
            "bias": bias, "gated": gated, "bs_last": bs_last}
    return dict(case, name=name) if name else case


def _adamw(name, tensors, times, dtype, bits, master=False):
    case = {"kind": "adamw", "tensors": tensors, "times": times, "dtype": dtype, "bits": bits, "master": master}
    return dict(case, name=name) if name else case


def listed():
    return [
        # what a 384-wide block's projection is given, kept for its backward pass: full batches, two interleaved blocks
        _quantize("quantize fp16 full", "1x192x2", "fp16", FULL),
        # feature-major rows that no vector divides
        _quantize("quantize fp32 last odd", "4x192x1", "fp32", 33 * 197, bs_last=True),
        # serving, one token: the gated projection of a 384-wide block
        _product("product fp16 one token", "1x768x192x2", "fp16", 1, act="silu", gated=True),
        # one image of 197 tokens (a class token makes them odd) through blocks of 64 inputs
        _product("product fp16 one image", "6x256x64x1", "fp16", 197, act="gelu", bias=True),
        # serving full batches
        _product("product fp16 full", "1x768x192x2", "fp16", FULL, act="silu", gated=True),
        # fp32 activations around dense 192 x 192 blocks, feature-major rows that no vector divides
        _product("product fp32 last odd", "4x192x192x1", "fp32", 33 * 197, act="gelu", bias=True, bs_last=True),
        # the training step of the 384-wide block's gated projection on full batches: the largest
        _product("train fp16 gated full", "1x768x192x2", "fp16", FULL, act="silu", gated=True, train=True),
        # training in fp32 on ten images, blocks that end inside 32 numbers
        _product("train fp32 odd", "2x96x72x3", "fp32", 10 * 197, act="gelu", bias=True, train=True),
        # the norms' weights and the gates of two 384-wide blocks: many small tensors
        _adamw("adamw fp16 vectors", "384,384,384", 2, "fp16", 32, master=True),
        # all parameters of twelve 384-wide blocks in fp32
        _adamw("adamw fp32 12 blocks", "589824,294912,24576,384,384,384", 12, "fp32", 32),
        # all parameters of four 768-wide blocks, moments in 8 bits, fp32 weights behind the fp16 ones
        _adamw("adamw fp16 4 blocks 8 bit", "2359296,1179648,49152,768,768,768", 4, "fp16", 8, master=True),
        # tensors that no block of 32 and no vector divides, moments in 8 bits, no weights behind them
        _adamw("adamw fp16 odd 8 bit", "30001,4097,385,33,1", 5, "fp16", 8),
    ]


def _numbers(text, sep="x"):
    return tuple(int(v) for v in text.split(sep))


def _lengths(case):
    return _numbers(case["tensors"], ",") * case["times"]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("quantize", "product", "product", "train", "adamw", "adamw"))
    dtype = rng.choice(("fp32", "fp16", "fp16"))
    if kind == "adamw":
        bits = rng.choice((8, 32))
        lengths = [_log(rng, 1, 1 << 21) for _ in range(rng.randint(1, 6))]
        lengths = [max(1, n // 32 * 32) if rng.random() < 0.6 else n for n in lengths]
        times = rng.randint(1, 30 // len(lengths) if bits == 8 else 24)
        case = _adamw(None, ",".join(map(str, lengths)), times, dtype, bits, dtype == "fp16" and rng.random() < 0.5)
        while _cost(case) > _cost(listed()[10]):
            case["times"] = (case["times"] + 1) // 2 if case["times"] > 1 else 1
            if case["times"] == 1:
                case["tensors"] = ",".join(str(max(1, n // 2)) for n in _numbers(case["tensors"], ","))
        return case
    batch = min(FULL, _log(rng, 1, FULL))
    bs_last = rng.random() < 0.4
    while True:
        c = rng.choice((16, 32, 48, 64, 96, 128, 192, 256, 384, 768))
        b = rng.choice((c, c, 2 * c, 4 * c, max(16, c // 4)))
        if rng.random() < 0.2:
            b += rng.randint(1, 15)
        if rng.random() < 0.2:
            c += rng.randint(1, 15)
        a, d = rng.choice((1, 1, 2, 3, 4, 6, 12)), rng.choice((1, 1, 2, 2, 3, 4, 6, 8, 16))
        if 64 <= a * d * max(b, c) <= 6144:
            break
    if kind == "quantize":
        return _quantize(None, "%dx%dx%d" % (a, c, d), dtype, batch, bs_last)
    gated = rng.random() < 0.4
    case = _product(None, "%dx%dx%dx%d" % (a, b, c, d), dtype, batch,
                    rng.choice(("silu", "gelu") if gated else ("none", "gelu")), rng.random() < 0.5, gated, bs_last,
                    kind == "train")
    while _cost(case) > _cost(listed()[6 if kind == "train" else 4]):
        case["batch"] = (case["batch"] + 1) // 2
    return case


def _cost(case):
    """Seconds of a pass at ordinary rates: what keeps drawn cases below the largest."""
    w = work(case)
    rate = 1e15 if case["kind"] == "product" else 6e13 if case["dtype"] == "fp32" else 3e14
    return w["bytes"] / 4e12 + w["flops"] / rate


class _Draws:
    """Values on the GPU from a seed."""

    def __init__(self, seed, dtype):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = dtype

    def normal(self, *shape, scale=1.0, mean=0.0, dtype=None):
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return (t * scale + mean).to(dtype or self.dtype)


def prepare(case, seed):
    """Inputs, weights, and for training the gradients of the results or the optimiser's state."""
    draws, dtype = _Draws(seed, DTYPES[case["dtype"]]), DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    if case["kind"] == "adamw":
        return _prepare_adamw(s, case, draws)
    batch, bs_last = case["batch"], case["bs_last"]

    def rows(features):
        return draws.normal(*((features, batch) if bs_last else (batch, features)))

    if case["kind"] == "quantize":
        a, c, d = _numbers(case["sizes"])
        s["x"] = rows(a * c * d)
        return s
    a, b, c, d = _numbers(case["pattern"])
    r = 2 * b if case["gated"] else b
    s["x"] = rows(a * c * d)
    factor = draws.normal(a * d * c, r, scale=1 / math.sqrt(c))
    s["bias"] = draws.normal(a * r * d, scale=0.1) if case["bias"] else None
    if case["kind"] == "product":
        # a program that serves keeps its weights as codes and scales
        s["codes"], s["scales"] = _pack(factor.float().view(a * d, c, r).transpose(1, 2).contiguous())
        return s
    s["factor"] = factor
    s["wanted"] = [s["x"], s["factor"]] + ([s["bias"]] if case["bias"] else [])
    s["grads"] = [rows(a * b * d)]
    for t in s["wanted"]:
        t.requires_grad_(True)
    return s


def _flat(lengths, dtype, make=None):
    """One buffer and the tensors in it, each from a multiple of 64 elements on."""
    starts, at = [], 0
    for n in lengths:
        starts.append(at)
        at += (n + 63) // 64 * 64
    buffer = torch.zeros(at, device="cuda", dtype=dtype)
    if make is not None:
        buffer.copy_(make(at))
    return buffer, [buffer[i:i + n] for i, n in zip(starts, lengths)]


def _prepare_adamw(s, case, draws):
    lengths, dtype = _lengths(case), DTYPES[case["dtype"]]
    s["all"], s["params"] = _flat(lengths, dtype, lambda n: draws.normal(n, scale=0.05))
    s["grads"] = _flat(lengths, dtype, lambda n: draws.normal(n, scale=1e-3 / GRAD_SCALE))[1]
    s["all_masters"], s["masters"] = None, None
    if case["master"]:  # weights that the fp16 ones are roundings of
        near = draws.normal(s["all"].numel(), scale=1e-4, dtype=torch.float32).clamp(-2e-4, 2e-4)
        s["all_masters"], s["masters"] = _flat(lengths, torch.float32, lambda n: s["all"].float() * (1 + near))
    m, ms = _flat(lengths, torch.float32, lambda n: draws.normal(n, scale=3e-4, dtype=torch.float32))
    v, vs = _flat(lengths, torch.float32, lambda n: draws.normal(n, scale=1e-3, dtype=torch.float32).square() + 1e-9)
    if case["bits"] == 32:
        s["all_moments"], s["m"], s["v"], s["scales"] = [m, v], ms, vs, None
        return s
    half = torch.full((), 0.5, device="cuda")
    packed = [_pack_moments(x, y, half, half) for x, y in zip(ms, vs)]
    s["m"], s["v"], s["scales"] = ([p[k] for p in packed] for k in range(3))
    return s


def run(state):
    case = state["case"]
    if own:
        return _RUN_OWN[case["kind"]](state, case)
    with torch.no_grad():
        return _RUN_PLAIN[case["kind"]](state, case)


# -- the framework's operators ---------------------------------------------------------------------


def _own_quantize(s, case):
    from ksmm_amd import quantize_mx

    return [quantize_mx(s["x"], _numbers(case["sizes"]), bs_last=case["bs_last"]).dequantize()]


def _own_product(s, case):
    from ksmm_amd import MXFactor, mx_linear

    w = MXFactor(s["codes"], s["scales"], _numbers(case["pattern"]), gated=case["gated"])
    return [mx_linear(s["x"], w, bias=s["bias"], act=case["act"], bs_last=case["bs_last"])]


def _own_train(s, case):
    from ksmm_amd import mx_linear

    y = mx_linear(s["x"], s["factor"], _numbers(case["pattern"]), bias=s["bias"], act=case["act"], gated=case["gated"],
                  bs_last=case["bs_last"])
    return [y.detach()] + list(torch.autograd.grad([y], s["wanted"], s["grads"]))


def _own_adamw(s, case):
    from ksmm_amd import adamw_moments, adamw_update

    adamw_update(s["params"], s["grads"], s["m"], s["v"], scales=s["scales"], masters=s["masters"], step=STEP, lr=LR,
                 betas=BETAS, eps=EPS, weight_decay=DECAY, grad_scale=GRAD_SCALE, seed=SEED)
    return _updated(s, case, adamw_moments(s["m"], s["v"], s["scales"]) if case["bits"] == 8 else None)


def _updated(s, case, moments):
    """The buffers that hold all tensors; moments in 8 bits as the values that they stand for."""
    out = [s["all"]] + ([s["all_masters"]] if case["master"] else [])
    return out + (s["all_moments"] if case["bits"] == 32 else [list(moments[0]), list(moments[1])])


_RUN_OWN = {"quantize": _own_quantize, "product": _own_product, "train": _own_train, "adamw": _own_adamw}


# -- in elementary operations, in 32 bits, rounded once (8-bit moments in 64: next to a border one bit decides) --------


def _exponent(top, below):
    """floor(log2 top) - below of each block's largest value, from LOWEST on."""
    e = torch.frexp(top)[1] - 1 - below
    return torch.where(top > 0, e, LOWEST).clamp(min=LOWEST)


def _power(e):
    """2 ** e in fp32, exactly."""
    return ((e + 127).to(torch.int32) << 23).view(torch.float32)


def _blocks(t):
    """(.., c) in blocks of 32, the last one filled with zeros."""
    t = torch.nn.functional.pad(t, (0, -t.shape[-1] % 32))
    return t.reshape(*t.shape[:-1], -1, 32)


def _round4(t):
    """(.., c) as 4-bit numbers: what each is of its block's power of two, and that power's exponent."""
    x = _blocks(t)
    e = _exponent(x.abs().amax(-1, keepdim=True), 2)
    y = x * _power(-e)
    size = y.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return torch.copysign((torch.round(size / step) * step).clamp(max=6), y), e


def _value4(t):
    q, e = _round4(t)
    return (q * _power(e)).flatten(-2)[..., :t.shape[-1]]


def _pack(t):
    """Codes (.., 16 bytes a block, the even places in the lower halves) and scales of (.., c)."""
    q, e = _round4(t)
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=t.device)
    code = torch.searchsorted(grid, q.abs()) | (q < 0).to(torch.int64) << 3
    pairs = code[..., 0::2] | code[..., 1::2] << 4
    return pairs.to(torch.uint8).flatten(-2), (e + 127).to(torch.uint8).squeeze(-1)


def _unpack(codes, scales, c):
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    grid = torch.cat([grid, -grid])
    both = torch.stack([codes & 15, codes >> 4], -1).to(torch.int64)
    values = grid[both].reshape(*scales.shape, 32) * _power(scales.to(torch.int32) - 127).unsqueeze(-1)
    return values.flatten(-2)[..., :c]


def _act(name, z):
    if name == "none":
        return z
    if name == "silu":
        return z * torch.sigmoid(z)
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))


def _act_slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "silu":
        g = torch.sigmoid(z)
        return g * (1 + z * (1 - g))
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _operand(t, a, k, d, case):
    """(a, d, n, k): what each block reads or writes, in fp32."""
    n, t = case["batch"], t.float()
    t = t.view(a, k, d, n).permute(0, 2, 3, 1) if case["bs_last"] else t.view(n, a, k, d).permute(1, 3, 0, 2)
    return t.contiguous()


def _tensor(t, case):
    """Blocks (a, d, n, k) in the layout of the tensors, in their type."""
    a, d, n, k = t.shape
    t = t.permute(0, 3, 1, 2).reshape(a * k * d, n) if case["bs_last"] else t.permute(2, 0, 3, 1).reshape(n, a * k * d)
    return t.to(DTYPES[case["dtype"]])


def _plain_quantize(s, case):
    a, c, d = _numbers(case["sizes"])
    return [_tensor(_value4(_operand(s["x"], a, c, d, case)), case)]


def _projections(s, case, x, w):
    """z, the first and the second half of it and the result; w (a, d, rows, c)."""
    a, b, c, d = _numbers(case["pattern"])
    r = w.shape[2]
    z = torch.matmul(x, w.transpose(2, 3).contiguous())
    if case["bias"]:
        z = z + s["bias"].float().view(a, r, d).permute(0, 2, 1).unsqueeze(2)
    g, u = (z[..., :b], z[..., b:]) if case["gated"] else (z, None)
    h = _act(case["act"], g)
    return g, u, h if u is None else h * u


def _plain_product(s, case):
    a, b, c, d = _numbers(case["pattern"])
    w = _unpack(s["codes"], s["scales"], c).view(a, d, -1, c)
    x = _value4(_operand(s["x"], a, c, d, case))
    return [_tensor(_projections(s, case, x, w)[2], case)]


def _plain_train(s, case):
    a, b, c, d = _numbers(case["pattern"])
    dtype = DTYPES[case["dtype"]]
    w = _value4(s["factor"].float().view(a, d, c, -1).transpose(2, 3).contiguous())
    x = _value4(_operand(s["x"], a, c, d, case))
    g, u, y = _projections(s, case, x, w)
    dz = _operand(s["grads"][0], a, b, d, case)
    if case["gated"]:
        dz = torch.cat([dz * u * _act_slope(case["act"], g), dz * _act(case["act"], g)], dim=3)
    else:
        dz = dz * _act_slope(case["act"], g)
    out = [_tensor(y, case), _tensor(torch.matmul(dz, w), case),
           torch.matmul(x.transpose(2, 3).contiguous(), dz).reshape(s["factor"].shape).to(dtype)]
    if case["bias"]:
        out.append(dz.sum(2).permute(0, 2, 1).reshape(-1).to(dtype))
    return out


def _mix(x):
    """32 bits, spread: (x ^ x >> 16) times 2^32 times the fraction of sqrt(2), the same with 15 and sqrt(3), x ^ x >> 16."""
    x = ((x ^ x >> 16) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ x >> 15) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ x >> 16


def _dither(n, tensor):
    """Two numbers in [0, 1) for each of a tensor's places, in steps of 2^-16."""
    key = _mix((_mix((SEED + tensor) & 0xFFFFFFFF) + STEP) & 0xFFFFFFFF)
    h = _mix(torch.arange(n, device="cuda") ^ key)
    return (h & 0xFFFF).float() / 65536, (h >> 16).float() / 65536


def _floor_to(y, dither, bits, least):
    """y >= 0 rounded down or up, as the dither says, to ``bits`` behind its leading one, from exponent ``least`` on."""
    q = torch.where(y > 0, torch.frexp(y)[1] - 1, least).clamp(min=least) - bits
    return torch.floor(y * _power(-q) + dither) * _power(q)


def _pack_moments(m, v, r, s):
    """e4m3 codes of m, e5m3 codes of v and the scales of both, (2, blocks of 32)."""
    n = m.numel()
    x, y = _blocks(m), _blocks(v)
    r, s = (_blocks(t) if t.dim() else t for t in (r, s))
    em, ev = _exponent(x.abs().amax(-1, keepdim=True), 7), _exponent(y.amax(-1, keepdim=True), 14)
    x, y = x * _power(-em), y * _power(-ev)
    x = torch.copysign(_floor_to(x.abs(), r, 3, -6), x)
    y = torch.where(y > 0, _floor_to(y, s, 3, -14).clamp(min=2.0 ** -17), 0.0)
    codes_m = x.float().to(torch.float8_e4m3fn).view(torch.uint8).flatten()[:n]
    codes_v = (y.float().to(torch.float16).view(torch.int16) >> 7).to(torch.uint8).flatten()[:n]
    scales = torch.stack([em.flatten() + 127, ev.flatten() + 127]).to(torch.uint8)
    return codes_m.contiguous(), codes_v.contiguous(), scales


def _unpack_moments(m, v, scales):
    n = m.numel()
    power = _power(scales.to(torch.int32) - 127).unsqueeze(-1)
    x = _blocks(m.view(torch.float8_e4m3fn).float()) * power[0]
    y = _blocks((v.to(torch.int16) << 7).view(torch.float16).float()) * power[1]
    return x.flatten()[:n], y.flatten()[:n]


def _step_of(case):
    """Of one step: what the weights keep, the rate, and what sqrt(v) is multiplied with."""
    return (1 - LR * DECAY, LR / (1 - BETAS[0] ** STEP), 1 / math.sqrt(1 - BETAS[1] ** STEP))


def _plain_adamw(s, case):
    keep, rate, root = _step_of(case)
    moments = [_plain_adamw_one(s, case, i, keep, rate, root) for i in range(len(s["params"]))]
    return _updated(s, case, ([m for m, _ in moments], [v for _, v in moments]))


def _plain_adamw_one(s, case, i, keep, rate, root):
    p, m, v = s["params"][i], s["m"][i], s["v"][i]
    w = s["masters"][i] if case["master"] else p.float()
    g = s["grads"][i].float() * GRAD_SCALE
    if case["bits"] == 8:
        m, v = (t.double() for t in _unpack_moments(m, v, s["scales"][i]))
        g = s["grads"][i].double() * GRAD_SCALE
    new_m = m * BETAS[0] + g * (1 - BETAS[0])
    new_v = v * BETAS[1] + g * g * (1 - BETAS[1])
    w = w * keep - rate * (new_m / (new_v.sqrt() * root + EPS))
    if case["master"]:
        s["masters"][i].copy_(w)
    p.copy_(w)
    if case["bits"] == 32:
        m.copy_(new_m)
        v.copy_(new_v)
        return m, v
    packed = _pack_moments(new_m, new_v, *_dither(m.numel(), i))
    for to, t in zip((s["m"][i], s["v"][i], s["scales"][i]), packed):
        to.copy_(t)
    return _unpack_moments(*packed)


_RUN_PLAIN = {"quantize": _plain_quantize, "product": _plain_product, "train": _plain_train, "adamw": _plain_adamw}


# -- from the definitions, in 64 bits ---------------------------------------------------------------


def exact(case, seed):
    with torch.no_grad():
        return {"quantize": _exact_quantize, "product": _exact_product, "train": _exact_product,
                "adamw": _exact_adamw}[case["kind"]](prepare(case, seed), case)


def _two(e):
    """2 ** e of whole e in 64 bits (powers and logarithms of the library may be a last bit off)."""
    return (e.to(torch.int64) + 1023 << 52).view(torch.float64)


def _level(t):
    """floor(log2 t); -300 where t is zero."""
    t = t.clamp(min=2.0 ** -300)
    e = torch.floor(torch.log2(t))
    return e + (_two(e + 1) <= t).double() - (_two(e) > t).double()


_MIDDLES = ((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0), (0.5, 0.5, 0.5, 0.5, 1.0, 1.0, 2.0))


def _nearest4(t):
    """The values of 4-bit numbers along the last axis: steps that |t| has passed, those in the middle to the even one."""
    out = torch.empty_like(t)
    for k in range(0, t.shape[-1], 32):
        x = t[..., k:k + 32]
        top = x.abs().amax(-1, keepdim=True)
        scale = _two(_level(top).sub(2).clamp(min=LOWEST))
        y, q = x.abs() / scale, torch.zeros_like(x)
        for i, (middle, step) in enumerate(zip(*_MIDDLES)):
            q += step * (y > middle if i % 2 == 0 else y >= middle)
        out[..., k:k + 32] = torch.sign(x) * q * scale
    return out


def _exact_quantize(s, case):
    a, c, d = _numbers(case["sizes"])
    x = s["x"].double()
    x = x.t() if case["bs_last"] else x
    x = _nearest4(x.reshape(-1, a, c, d).transpose(2, 3)).transpose(2, 3).reshape(x.shape)
    return [x.t() if case["bs_last"] else x]


def _exact_weights(s, case, block):
    """(c, rows) of one block."""
    a, b, c, d = _numbers(case["pattern"])
    if case["kind"] == "train":
        return _nearest4(s["factor"].detach().double()[block * c:(block + 1) * c].t()).t()
    codes, e = s["codes"][block].long(), s["scales"][block].double() - 127
    w = e.new_zeros(codes.shape[0], codes.shape[1] * 2)
    for half in (0, 1):
        code = (codes >> 4 * half) & 15
        power, odd = (code & 7) // 2, (code & 1).double()
        size = torch.where(power == 0, odd / 2, (1 + odd / 2) * _two(power - 1))
        w[:, half::2] = torch.where(code >= 8, -size, size)
    return (w * _two(e).repeat_interleave(32, 1))[:, :c].t()


def _exact_product(s, case):
    """Block by block: its rows and columns of the sparse matrices."""
    a, b, c, d = _numbers(case["pattern"])
    train, gated, last = case["kind"] == "train", case["gated"], case["bs_last"]
    r = 2 * b if gated else b
    x = s["x"].detach().double()
    x = x.t() if last else x
    n = x.shape[0]
    y = x.new_empty(n, a * b * d)
    bias = s["bias"].detach().double() if case["bias"] else None
    if train:
        dy = s["grads"][0].double()
        dy = dy.t() if last else dy
        dx, dfactor, dbias = torch.empty_like(x), x.new_empty(s["factor"].shape), x.new_empty(a * r * d)
    for i in range(a):
        for l in range(d):
            cols = torch.arange(c, device=x.device) * d + i * c * d + l
            outs = torch.arange(b, device=x.device) * d + i * b * d + l
            terms = torch.arange(r, device=x.device) * d + i * r * d + l
            w, xi = _exact_weights(s, case, i * d + l), _nearest4(x[:, cols])
            z = xi @ w
            if bias is not None:
                z = z + bias[terms]
            g = z[:, :b]
            if case["act"] == "none":
                value, slope = g, torch.ones_like(g)
            else:
                phi = torch.reciprocal(1 + torch.exp(-g)) if case["act"] == "silu" else torch.special.ndtr(g)
                slope = phi + g * (phi * (1 - phi) if case["act"] == "silu" else torch.exp(-g * g / 2) / math.sqrt(2 * math.pi))
                value = g * phi
            y[:, outs] = value * z[:, b:] if gated else value
            if not train:
                continue
            dz = dy[:, outs]
            dz = torch.cat([dz * z[:, b:] * slope, dz * value], 1) if gated else dz * slope
            dx[:, cols] = dz @ w.t()
            dfactor[(i * d + l) * c:(i * d + l + 1) * c] = xi.t() @ dz
            dbias[terms] = dz.sum(0)
    if not train:
        return [y.t() if last else y]
    return [y.t() if last else y, dx.t() if last else dx, dfactor] + ([dbias] if case["bias"] else [])


def _exact_adamw(s, case):
    beta1, beta2 = BETAS
    lengths = _lengths(case)
    out = {k: [] for k in ("w", "m", "v")}
    for i, n in enumerate(lengths):
        g = s["grads"][i].double() * GRAD_SCALE
        w = (s["masters"] if case["master"] else s["params"])[i].double()
        m, v = s["m"][i], s["v"][i]
        if case["bits"] == 8:
            at = torch.arange(n, device="cuda") // 32
            scale = _two(s["scales"][i].long() - 127)
            sign, e, f = m >> 7, (m >> 3 & 15).double(), (m & 7).double()
            m = torch.where(e > 0, (8 + f) * _two(e - 10), f * 2.0 ** -9) * torch.where(sign > 0, -1.0, 1.0) * scale[0][at]
            e, f = (v >> 3).double(), (v & 7).double()
            v = torch.where(e > 0, (8 + f) * _two(e - 18), f * 2.0 ** -17) * scale[1][at]
        m, v = beta1 * m.double() + (1 - beta1) * g, beta2 * v.double() + (1 - beta2) * g ** 2
        hat_m, hat_v = m / (1 - beta1 ** STEP), v / (1 - beta2 ** STEP)
        out["w"].append(w - LR * DECAY * w - LR * hat_m / (hat_v ** 0.5 + EPS))
        if case["bits"] == 8:
            r, t = (d.double() for d in _dither(n, i))
            m, v = _exact_rounded(m, r, at, 7, -6, False), _exact_rounded(v, t, at, 14, -14, True)
        out["m"].append(m)
        out["v"].append(v)
    if case["bits"] == 8:
        w = _spread(out["w"], s["all"])
        return [w] + ([w] if case["master"] else []) + [out["m"], out["v"]]
    # (gaps between the tensors are not touched)
    w = _spread(out["w"], s["all"])
    masters = [_spread(out["w"], s["all_masters"])] if case["master"] else []
    return [w] + masters + [_spread(out[k], t) for k, t in zip(("m", "v"), s["all_moments"])]


def _spread(parts, like):
    """Tensors in a buffer, each from a multiple of 64 elements on; what is between them as it was."""
    out, at = like.double(), 0
    for t in parts:
        out[at:at + t.numel()] = t
        at += (t.numel() + 63) // 64 * 64
    return out


def _exact_rounded(t, dither, at, below, least, positive):
    top = torch.zeros(int(at[-1]) + 1, dtype=t.dtype, device=t.device).scatter_reduce(0, at, t.abs(), "amax")
    scale = _two((_level(top) - below).clamp(min=LOWEST))[at]
    y = t.abs() / scale
    step = _two(_level(y).clamp(min=least) - 3)
    q = torch.floor(y / step + dither) * step
    if positive:
        q = torch.where(y > 0, q.clamp(min=2.0 ** (least - 3)), q)
    return torch.sign(t) * q * scale


def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "adamw":
        n = sum(_lengths(case))
        # gradient and weight read, weight written, masters and moments both; what the 8-bit ones stand for is written too
        moments = 16 if case["bits"] == 32 else 4 + 0.125 + 8
        return {"bytes": n * (3 * size + (8 if case["master"] else 0) + moments), "flops": 16 * n}
    if case["kind"] == "quantize":
        a, c, d = _numbers(case["sizes"])
        n = case["batch"] * a * c * d
        # codes and scales are written and read again
        return {"bytes": n * (2 * size + 2 * 17 / 32), "flops": 8 * n}
    a, b, c, d = _numbers(case["pattern"])
    r = 2 * b if case["gated"] else b
    weights, bias, values = a * r * c * d, a * r * d if case["bias"] else 0, case["batch"] * a * d * (b + c)
    if case["kind"] == "product":
        return {"bytes": weights * 17 / 32 + size * (bias + values), "flops": 2 * case["batch"] * weights}
    return {"bytes": 2 * size * (weights + bias + values), "flops": 6 * case["batch"] * weights}
