"""What the C ABI of the 4-bit products and of AdamW refuses before anything is launched (no GPU)."""
import ctypes

import pytest
import torch

from tests import mx_ref as R

NULL, PATTERN, BATCH, DTYPE, LARGE, ALGO, WORKSPACE, ALIAS, EPILOGUE = -1, -2, -3, -4, -5, -6, -9, -11, -12
FAR = [(i + 1) << 32 for i in range(16)]  # addresses that are never touched: every call here is refused


def test_sizes(lib):
    assert lib.ksmm_mx_blocks(7, 2, 33, 3) == 7 * 2 * 2 * 3
    assert lib.ksmm_mx_blocks(1, 1, 32, 1) == 1
    assert lib.ksmm_mx_blocks(0, 1, 32, 1) == BATCH
    assert lib.ksmm_mx_blocks(1, 1, 0, 1) == PATTERN
    assert lib.ksmm_mx_blocks(1 << 31, 1, 1, 1) == LARGE


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("bs_last", [0, 1])
def test_conversions_refuse(lib, back, bs_last):
    rows, a, c, d = 10, 2, 40, 3
    x, codes, scales = FAR[:3]
    blocks = rows * a * d * 2

    def call(x=x, codes=codes, scales=scales, rows=rows, a=a, c=c, d=d, dtype=1):
        if back:
            return lib.ksmm_mx_dequantize(codes, scales, x, rows, a, c, d, dtype, bs_last, None)
        return lib.ksmm_mx_quantize(x, codes, scales, rows, a, c, d, dtype, bs_last, None)

    for k in ("x", "codes", "scales"):
        assert call(**{k: None}) == NULL
    assert call(rows=0) == BATCH and call(a=0) == PATTERN and call(c=0) == PATTERN and call(d=-1) == PATTERN
    assert call(dtype=2) == DTYPE and call(dtype=7) == DTYPE
    assert call(rows=1 << 30) == LARGE
    assert call(codes=codes + 8) == WORKSPACE
    size = 2 * rows * a * c * d
    assert call(codes=x + (size - 1) // 16 * 16) == ALIAS and call(scales=x + size - 1) == ALIAS
    assert call(x=codes + 16 * blocks - 1) == ALIAS and call(scales=codes + 16 * blocks - 1) == ALIAS


@pytest.mark.parametrize("bs_last", [0, 1])
def test_values_of_both_operands_refuse(lib, bs_last):
    batch, rows, a, c, d = 10, 7, 2, 40, 3
    names = ["x_codes", "x_scales", "x", "w_codes", "w_scales", "w"]
    at = dict(zip(names, FAR))

    def call(batch=batch, rows=rows, a=a, c=c, d=d, dtype=1, **change):
        p = dict(at, **change)
        return lib.ksmm_mx_values(*(p[k] for k in names), batch, rows, a, c, d, dtype, bs_last, None)

    for k in names:
        assert call(**{k: None}) == NULL
    assert call(batch=0) == BATCH and call(rows=0) == BATCH and call(a=0) == PATTERN and call(d=0) == PATTERN and call(dtype=2) == DTYPE
    assert call(batch=1 << 30) == LARGE and call(rows=1 << 30) == LARGE and call(a=1 << 20, d=1 << 20, c=1) == LARGE
    assert call(x_codes=at["x_codes"] + 8) == WORKSPACE and call(w_codes=at["w_codes"] + 4) == WORKSPACE
    sizes = {"x_codes": batch * a * d * 32, "x_scales": batch * a * d * 2, "w_codes": rows * a * d * 32, "w_scales": rows * a * d * 2}
    for out, other in (("x", "w"), ("w", "x")):
        for k in sizes:
            assert call(**{out: at[k] + sizes[k] - 1}) == ALIAS
        assert call(**{out: at[other] + 2}) == ALIAS


@pytest.mark.parametrize("c", [40, 9000])
def test_products_refuse(lib, c):
    n, a, b, d = 9, 2, 24, 3
    names = ["x", "x_scales", "w", "w_scales", "bias", "y", "codes", "scales", "workspace"]
    at = dict(zip(names, FAR))
    for dtype, size in ((0, 4), (1, 2)):
        for gated in (0, 1):
            for bs_last in (0, 1):
                need = lib.ksmm_mx_forward_workspace(n, a, b, c, d, dtype, bs_last, gated)
                assert (need > 0) == (c == 9000)

                def call(quantised, bytes=need, act=0, n=n, a=a, b=b, c=c, d=d, dtype=dtype, gated=gated, **change):
                    p = dict(at, **change)
                    return lib.ksmm_mx_forward(p["x"], p["x_scales"] if quantised else None, p["w"], p["w_scales"], p["bias"], p["y"], p["codes"], p["scales"], p["workspace"], bytes, n, a, b, c, d,
                                               dtype, bs_last, act, gated, None)

                for q in (False, True):
                    for k in ("x", "w", "w_scales", "y"):
                        assert call(q, **{k: None}) == NULL
                    assert call(q, n=0) == BATCH and call(q, b=0) == PATTERN and call(q, dtype=2) == DTYPE
                    assert call(q, b=1 << 30) == LARGE and call(q, n=0x7fffffff) == LARGE and call(q, act=3) == EPILOGUE
                    if not gated:
                        assert call(q, act=2) == EPILOGUE
                    assert call(q, w=at["w"] + 8) == WORKSPACE
                    rows = b * (1 + gated)
                    blocks = (c + 31) // 32 * a * d
                    sizes = {"x": n * blocks * 16 if q else n * a * c * d * size, "x_scales": n * blocks, "w": rows * blocks * 16, "w_scales": rows * blocks,
                             "bias": a * rows * d * size}
                    for k in sizes:
                        if k != "x_scales" or q:
                            assert call(q, y=at[k] + sizes[k] - 1) == ALIAS, (q, k)
                            if not q:  # (codes that are given are not written)
                                assert call(q, codes=(at[k] + sizes[k] - 1) // 16 * 16) == ALIAS and call(q, scales=at[k] + sizes[k] - 1) == ALIAS, k
                assert call(False, codes=None) == NULL and call(False, scales=None) == NULL and call(False, codes=at["codes"] + 8) == WORKSPACE
                assert call(False, codes=at["y"]) == ALIAS and call(False, scales=at["codes"]) == ALIAS
                assert call(True, x=at["x"] + 4) == WORKSPACE
                if need:
                    assert call(False, bytes=need - 1) == WORKSPACE and call(False, workspace=None) == WORKSPACE and call(False, workspace=at["workspace"] + 4) == WORKSPACE
                    for k in ("x", "w", "w_scales", "bias", "y"):
                        assert call(False, workspace=at[k]) == ALIAS


@pytest.mark.parametrize("gated", [0, 1])
@pytest.mark.parametrize("dtype", [0, 1])
def test_slopes_refuse(lib, dtype, gated):
    n, a, b, c, d, size = 9, 2, 24, 40, 1, (4, 2)[dtype]
    names = ["x", "x_scales", "w", "w_scales", "bias", "dy", "dz"]
    at = dict(zip(names, FAR))

    def call(n=n, a=a, b=b, c=c, d=d, dtype=dtype, bs_last=0, act=1, **change):
        p = dict(at, **change)
        return lib.ksmm_mx_slope(*(p[k] for k in names), n, a, b, c, d, dtype, bs_last, act, gated, None)

    for k in ("x", "x_scales", "w", "w_scales", "dy"):
        assert call(**{k: None}) == NULL
    assert call(n=0) == BATCH and call(c=0) == PATTERN and call(dtype=2) == DTYPE and call(n=0x7fffffff) == LARGE and call(act=3) == EPILOGUE
    if not gated:
        assert call(act=0) == EPILOGUE and call(act=2) == EPILOGUE
    assert call(w=at["w"] + 8) == WORKSPACE and call(x=at["x"] + 4) == WORKSPACE
    rows = b * (1 + gated)
    sizes = {"x": n * a * 2 * 16, "x_scales": n * a * 2, "w": rows * a * 2 * 16, "w_scales": rows * a * 2, "bias": a * rows * size, "dy": n * a * b * size}
    for k in sizes:
        assert call(dz=at[k] + sizes[k] - 1) == ALIAS, k
    # what there is a kernel for is said without a launch
    for bs_last in (0, 1):
        assert call(dz=None, bs_last=bs_last) == 0
        assert call(dz=None, bs_last=bs_last, d=2) == 0 and call(dz=None, bs_last=bs_last, d=3) == (0 if bs_last or dtype == 1 else ALGO)
        assert call(dz=None, bs_last=bs_last, d=5) == (0 if bs_last else ALGO) and call(dz=None, bs_last=bs_last, c=2000) == ALGO
        assert call(bs_last=bs_last, c=2000) == ALGO


def table(count=2, n=100, small=True, master=True):
    from ksmm_amd._lib import KsmmAdamwTensor

    t = (KsmmAdamwTensor * count)()
    for i in range(count):
        p = [(8 * i + k + 1) << 32 for k in range(6)]
        t[i] = KsmmAdamwTensor(p[0], p[1], p[2] if master else None, p[3], p[4], p[5] if small else None, n)
    return t


def desc(bits=8, **change):
    from ksmm_amd._lib import KsmmAdamwDesc

    v = dict(dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, grad_scale=1.0, step=1, device_step=None, seed=0, bits=bits, follow=0), **change)
    return KsmmAdamwDesc(*(v[k] for k, _ in KsmmAdamwDesc._fields_))


@pytest.mark.parametrize("bits", [8, 32])
def test_steps_refuse(lib, bits):
    def call(d=None, t=None, count=2, dtype=1):
        return lib.ksmm_adamw_update(ctypes.byref(d or desc(bits)), t if t is not None else table(), count, dtype, None)

    nan, inf = float("nan"), float("inf")
    for change in (dict(beta1=1.0), dict(beta2=1.0), dict(beta1=-0.1), dict(beta2=nan), dict(lr=inf), dict(eps=nan), dict(eps=1e-38), dict(weight_decay=inf), dict(grad_scale=nan), dict(step=0),
                   dict(step=-5)):
        assert call(desc(bits, **change)) == ALGO, change
    assert call(desc(16)) == DTYPE and call(dtype=2) == DTYPE and call(count=-1) == BATCH
    assert lib.ksmm_adamw_update(None, table(), 2, 1, None) == NULL and lib.ksmm_adamw_update(ctypes.byref(desc(bits)), None, 2, 1, None) == NULL
    for k in ("weight", "grad", "m", "v"):
        t = table()
        setattr(t[1], k, None)
        assert call(t=t) == NULL
    t = table()
    t[1].master = None
    assert call(t=t) == NULL  # (masters for all or for none)
    t = table()
    t[1].scales = None
    if bits == 8:
        assert call(t=t) == NULL
    for n, error in ((-1, BATCH), (1 << 31, LARGE)):
        t = table()
        t[0].n = n
        assert call(t=t) == error
    # nothing that is written may overlap anything else, of its own tensor or of another
    size = {"weight": 200, "grad": 200, "master": 400, "m": 100 if bits == 8 else 400, "v": 100 if bits == 8 else 400, "scales": 8}
    written = ["weight", "master", "m", "v"] + (["scales"] if bits == 8 else [])
    for w in written:
        for other in size:
            if other == "scales" and bits == 32:
                continue
            for i in (0, 1):
                if (i, other) == (0, w):
                    continue
                t = table()
                setattr(t[0], w, getattr(t[i], other) + size[other] - 1)
                assert call(t=t) == ALIAS, (w, other, i)
    t = table()
    assert call(desc(bits, device_step=t[0].m + 8), t) == ALIAS


def test_moments_refuse(lib):
    from ksmm_amd._lib import KsmmAdamwMoment

    def made(**change):
        t = (KsmmAdamwMoment * 2)()
        for i in range(2):
            t[i] = KsmmAdamwMoment(*((8 * i + k + 1) << 32 for k in range(5)), 100)
        for k, v in change.items():
            setattr(t[1], k, v)
        return t

    for k in ("m", "v", "scales", "m_out", "v_out"):
        assert lib.ksmm_adamw_moments(made(**{k: None}), 2, None) == NULL
    base = made()
    for o in ("m_out", "v_out"):
        for k in ("m", "v", "scales"):
            assert lib.ksmm_adamw_moments(made(**{o: getattr(base[0], k)}), 2, None) == ALIAS
    assert lib.ksmm_adamw_moments(made(v_out=base[0].m_out + 396), 2, None) == ALIAS
    assert lib.ksmm_adamw_moments(made(n=-1), 2, None) == BATCH and lib.ksmm_adamw_moments(made(n=1 << 31), 2, None) == LARGE
    assert lib.ksmm_adamw_moments(None, 2, None) == NULL and lib.ksmm_adamw_moments(made(), -1, None) == BATCH
    assert lib.ksmm_adamw_moments(None, 0, None) == 0


def test_the_hash_is_even():
    """Means of 65536 numbers in [0, 1) of consecutive places, steps and tensors: 0.5 within five deviations of 0.29 / 256."""
    for seed, tensor, step in ((0, 0, 1), (0, 0, 2), (0, 1, 1), (7, 3, 1000), (123456789, 0, 5)):
        for r in R.dither(65536, seed, tensor, step):
            assert abs(float(r.mean()) - 0.5) <= 5 * 0.29 / 256
            assert abs(float((r[1:] * r[:-1]).mean()) - 0.25) <= 5 * 0.23 / 256  # neighbours
    a, b = R.dither(65536, 0, 0, 1), R.dither(65536, 0, 0, 2)
    for x, y in ((a[0], a[1]), (a[0], b[0]), (a[0], R.dither(65536, 0, 1, 1)[0])):
        assert abs(float(((x - 0.5) * (y - 0.5)).mean())) <= 5 / 12 / 256


def test_modules_refuse():
    from ksmm_amd import KSLinearMX, MXLinear, adamw_update, quantize_mx

    with pytest.raises(AssertionError):
        KSLinearMX([(1, 4, 4, 1)], dtype=torch.float8_e4m3fn)
    with pytest.raises(RuntimeError):
        quantize_mx(torch.zeros(2, 4), (1, 4, 1))
    with pytest.raises(ValueError):
        MXLinear.of(torch.nn.Linear(2, 2))
    with pytest.raises((RuntimeError, ValueError)):
        adamw_update([torch.zeros(2)], [torch.zeros(2)], [torch.zeros(2)], [torch.zeros(2)])


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("c,d", [(40, 1), (40, 5), (9000, 1)])
def test_sums_refuse(lib, c, d, dtype):
    n, a, b, size = 9, 2, 24, (4, 2)[dtype]
    names = ["x", "x_scales", "w", "w_scales", "bias", "z"]
    at = dict(zip(names, FAR))

    def call(n=n, a=a, b=b, c=c, d=d, dtype=dtype, bs_last=0, **change):
        p = dict(at, **change)
        return lib.ksmm_mx_sums(*(p[k] for k in names), n, a, b, c, d, dtype, bs_last, None)

    for bs_last in (0, 1):
        for k in ("x", "x_scales", "w", "w_scales", "z"):
            assert call(bs_last=bs_last, **{k: None}) == NULL
        assert call(bs_last=bs_last, n=0) == BATCH and call(bs_last=bs_last, b=0) == PATTERN and call(bs_last=bs_last, dtype=2) == DTYPE
        assert call(bs_last=bs_last, n=0x7fffffff) == LARGE and call(bs_last=bs_last, w=at["w"] + 8) == WORKSPACE and call(bs_last=bs_last, x=at["x"] + 4) == WORKSPACE
        blocks = (c + 31) // 32 * a * d
        sizes = {"x": n * blocks * 16, "x_scales": n * blocks, "w": b * blocks * 16, "w_scales": b * blocks, "bias": a * b * d * size}
        for k in sizes:
            assert call(bs_last=bs_last, z=at[k] + sizes[k] - 1) == ALIAS, k
        assert call(bs_last=bs_last, z=at["x"] - size * n * a * b * d + 1) == ALIAS
