"""AdamW over many tensors (adamw_update, adamw_moments, KSAdamW) against the formula in float64.

Tolerances.  Moments in 8 bits: the codes are equal, as both sides compute them in 64 bits.  fp32 values are results of at most eight
roundings of 2^-24 each of terms no larger than theirs, but for m, where gradient and momentum may cancel: against the largest
magnitudes of the operands, elementwise 1e-6.  fp16 weights: half a step, 2^-11 of the value or 3e-8, on top of that."""
import pytest
import torch

from tests import mx_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16}
HOW = dict(lr=3e-3, betas=(0.9, 0.995), eps=1e-8, weight_decay=0.02, grad_scale=0.25)


def make(lengths, prec, bits, master, seed=0, off=0):
    """Parameters, gradients and state; ``off``: values before each tensor, so that none is aligned."""
    g = torch.Generator().manual_seed(seed)

    def place(t):
        room = torch.empty(t.numel() + off, dtype=t.dtype, device="cuda")
        room[off:].copy_(t)
        return room[off:]

    s = {"w": [], "g": [], "m": [], "v": [], "scales": [] if bits == 8 else None, "master": [] if master else None}
    for n in lengths:
        w = torch.randn(n, generator=g) * 0.1
        s["w"].append(place(w.to(DT[prec])))
        if master:
            s["master"].append(place(w.to(DT[prec]).float() * (1 + 1e-4 * torch.rand(n, generator=g))))
        s["g"].append(place((torch.randn(n, generator=g) * torch.exp2(torch.randint(-8, 3, (n,), generator=g).float())).to(DT[prec])))
        m, v = torch.randn(n, generator=g) * 0.1, torch.randn(n, generator=g).square() * torch.exp2(torch.randint(-20, 2, (n,), generator=g).float())
        if bits == 8:
            half = torch.full((n,), 0.5).double()
            cm, cv, sc = R.encode_moments(m.double(), v.double(), half, half)
            s["m"].append(place(cm)), s["v"].append(place(cv)), s["scales"].append(sc.cuda())
        else:
            s["m"].append(place(m)), s["v"].append(place(v))
    return s


def close(x, y, size, dtype):
    """Whether x is y within 1e-6 of ``size`` and what its type takes."""
    x = x.double().cpu()
    room = 1e-6 * size + (y.abs() * 2.0 ** -11 + 3.1e-8 if dtype == torch.float16 else 1e-38)
    return bool(((x - y).abs() <= room).all())


def check(lengths, prec, bits, master, step=7, seed=3, off=0, steps=2):
    from ksmm_amd import adamw_moments, adamw_update

    s = make(lengths, prec, bits, master, off=off)
    for t in range(step, step + steps):
        before = [[x.clone() for x in s[k]] if s[k] is not None else None for k in ("w", "m", "v", "scales", "master")]
        adamw_update(s["w"], s["g"], s["m"], s["v"], s["scales"], s["master"], step=t, seed=seed, **HOW)
        decoded = adamw_moments(s["m"], s["v"], s["scales"]) if bits == 8 else None
        for i, n in enumerate(lengths):
            w, m, v, sc, ma = (x[i] if x is not None else None for x in before)
            m, v = R.decode_moments(m, v, sc) if bits == 8 else (m.cpu().double(), v.cpu().double())
            w0 = (ma if master else w).cpu().double()
            w1, m1, v1 = R.adamw(w0, s["g"][i], m, v, t, HOW["lr"], HOW["betas"], HOW["eps"], HOW["weight_decay"], HOW["grad_scale"])
            # (what m is a difference of, at the rate that it is taken with)
            apart = R.adamw(torch.zeros_like(w0), s["g"][i].abs(), m.abs(), v, t, HOW["lr"], HOW["betas"], HOW["eps"], 0.0, HOW["grad_scale"])[0].abs()
            size = w0.abs() + apart
            assert close(s["w"][i], w1, size, DT[prec])
            if master:
                assert close(s["master"][i], w1, size, torch.float32)
                assert torch.equal(s["w"][i], s["master"][i].to(DT[prec]))
            if bits == 32:
                assert close(s["m"][i], m1, m.abs() + s["g"][i].cpu().double().abs(), torch.float32) and close(s["v"][i], v1, v1, torch.float32)
                continue
            cm, cv, sc1 = R.encode_moments(m1, v1, *R.dither(n, seed, i, t))
            assert torch.equal(s["scales"][i].cpu(), sc1)
            x, y = R.decode_moments(cm, cv, sc1)
            for got, want in zip(R.decode_moments(s["m"][i], s["v"][i], s["scales"][i]), (x, y)):
                assert torch.equal(got, want)
            assert torch.equal(decoded[0][i].cpu().double(), x) and torch.equal(decoded[1][i].cpu().double(), y)
            # a step of the type at most from the moment itself, and nothing above zero is lost
            power = torch.exp2(sc1.double() - 127).repeat_interleave(32, 1)[:, :n]
            assert bool(((x - m1).abs() <= torch.maximum(m1.abs() / 8, power[0] * 2.0 ** -9)).all())
            assert bool(((y - v1).abs() <= torch.maximum(v1 / 8, power[1] * 2.0 ** -17)).all()) and bool((y[v1 > 0] > 0).all())


LENGTHS = [[1], [7, 8, 9, 31, 32, 33, 0, 64], [4096, 4097, 1, 12345], [50000]]


@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
@pytest.mark.parametrize("lengths", LENGTHS)
def test_steps(lengths, prec, bits, master, off):
    check(lengths, prec, bits, master, off=off)


@pytest.mark.parametrize("bits", [8, 32])
def test_more_tensors_than_a_launch_takes(bits):
    check([1 + 17 * i % 90 for i in range(200)], "fp16", bits, True, steps=1)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("step", [1, 2, 100000])
def test_first_and_late_steps(bits, step):
    check([300, 40], "fp32", bits, False, step=step, steps=1)


def test_zeros_are_a_state_to_start_from():
    from ksmm_amd import adamw_moments, adamw_update

    n = 100
    w, g = torch.zeros(n, device="cuda"), torch.linspace(-1, 1, n).cuda()
    m, v, s = (torch.zeros(k, dtype=torch.uint8, device="cuda") for k in (n, n, 8))
    adamw_update([w], [g], [m], [v], [s.view(2, 4)], lr=0.1, weight_decay=0.0, betas=(0.9, 0.999))
    # the first step is one of length lr against the gradient's sign, whatever its size
    assert float((w + 0.1 * g.sign()).abs().max()) <= 1e-6
    adamw_update([w], [torch.zeros_like(g)], [m], [v], [s.view(2, 4)], step=2)
    assert torch.isfinite(adamw_moments([m], [v], [s.view(2, 4)])[1][0]).all()
    # a block without a gradient keeps zeros
    m, v, s = (torch.zeros(k, dtype=torch.uint8, device="cuda") for k in (n, n, 8))
    before = w.clone()
    adamw_update([w], [torch.zeros_like(g)], [m], [v], [s.view(2, 4)], weight_decay=0.0)
    assert torch.equal(w, before) and not m.any() and not v.any()


@pytest.mark.parametrize("bits", [8, 32])
def test_infinities_and_nans_reach_their_element_alone(bits):
    from ksmm_amd import adamw_moments, adamw_update

    s, clean = make([70], "fp32", bits, False), make([70], "fp32", bits, False)
    bad = [3, 40, 69]
    for i, x in zip(bad, (float("nan"), float("inf"), -1e30)):
        s["g"][0][i] = x
        clean["g"][0][i] = 0.0
    rest = torch.ones(70, dtype=torch.bool)
    rest[bad] = False
    for t in (5, 6):
        for k in (s, clean):
            adamw_update(k["w"], k["g"], k["m"], k["v"], k["scales"], step=t, **HOW)
        if bits == 32:
            assert torch.equal(s["w"][0][rest], clean["w"][0][rest])
        assert torch.isnan(s["w"][0][bad[:2]]).all() and torch.isfinite(s["w"][0][rest]).all()
    if bits == 8:
        m, v = adamw_moments(s["m"], s["v"], s["scales"])
        assert torch.isnan(m[0][bad[:2]]).all() and torch.isfinite(m[0][rest]).all() and torch.isfinite(v[0][rest]).all()


def test_moments_in_8_bits_keep_their_mean():
    """1000 steps of one gradient size: v of 2000 elements in the mean as in 32 bits.  An element's v wanders: the variance of a step is
    f (1 - f) of a step of the type squared (an eighth of the value at most), f the share of it that a step of v moves; with
    1 - beta2 = 0.01 it stays below 0.01 / 8 of the square and its sum over the memory of 1 / (2 * 0.01) steps below 0.0625: a
    deviation of a quarter at most, of the mean of 2000 elements a hundredth of it, 6e-3; four of these."""
    from ksmm_amd import adamw_moments, adamw_update

    n = 2000
    g = torch.Generator().manual_seed(0)
    w = torch.zeros(n, device="cuda")
    m, v, s = (torch.zeros(k, dtype=torch.uint8, device="cuda") for k in (n, n, 2 * 63))
    s = s.view(2, 63)
    want = torch.zeros(n).double()
    for t in range(1, 1001):
        grad = torch.randn(n, generator=g).sign() * 0.3
        adamw_update([w], [grad.cuda()], [m], [v], [s], step=t, betas=(0.9, 0.99), lr=1e-4)
        want = 0.99 * want + 0.01 * grad.double().square()
    got = adamw_moments([m], [v], [s])[1][0].cpu().double()
    assert abs(float(got.mean() / want.mean()) - 1) <= 0.024


def test_follow():
    from ksmm_amd import adamw_update

    s = make([100], "fp16", 32, True)
    s["w"][0][:10] = 2.0  # written by somebody else
    before = s["master"][0].clone()
    adamw_update(s["w"], s["g"], s["m"], s["v"], None, s["master"], follow=True, lr=0.0)
    assert torch.equal(s["master"][0][10:], before[10:]) and bool((s["master"][0][:10] == 2.0).all())


def test_refusals():
    from ksmm_amd import KSAdamW, adamw_moments, adamw_update
    from ksmm_amd._lib import KsmmError

    s = make([64, 64], "fp32", 32, False)
    e = make([64, 64], "fp32", 8, False)
    args = s["w"], s["g"], s["m"], s["v"]
    for how in (dict(step=0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(lr=float("nan")), dict(eps=float("inf")), dict(grad_scale=float("inf")),
                dict(masters=s["w"][:1]), dict(scales=e["scales"]), dict(step=torch.ones(1, device="cuda")), dict(step=torch.ones(1, dtype=torch.int64))):
        with pytest.raises((ValueError, RuntimeError)):
            adamw_update(*args, **how)
    with pytest.raises(ValueError):
        adamw_update(s["w"], s["g"][:1], s["m"], s["v"])
    with pytest.raises(ValueError):
        adamw_update(s["w"], [g.half() for g in s["g"]], s["m"], s["v"])
    with pytest.raises(AssertionError):
        adamw_update([w.double() for w in s["w"]], s["g"], s["m"], s["v"])
    with pytest.raises(RuntimeError):
        adamw_update([w.cpu() for w in s["w"]], s["g"], s["m"], s["v"])
    with pytest.raises(RuntimeError):
        adamw_update([w.view(8, 8).t() for w in s["w"]], s["g"], s["m"], s["v"])
    with pytest.raises(ValueError):
        adamw_moments(e["m"], e["v"], [x[:, :1].contiguous() for x in e["scales"]])
    # a tensor twice, a state for two, a gradient in a state
    for w, g, m, v in (((s["w"][0],) * 2, s["g"], s["m"], s["v"]), (s["w"], s["g"], (s["m"][0],) * 2, s["v"]), (s["w"], s["m"], s["m"], s["v"])):
        with pytest.raises(KsmmError):
            adamw_update(list(w), list(g), list(m), list(v))
    adamw_update(s["w"], [s["g"][0]] * 2, s["m"], s["v"])  # (one gradient for two is fine)
    adamw_update([], [], [], [])
    p = torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))
    for call in (lambda: KSAdamW([p], bits=4), lambda: KSAdamW([p], betas=(0.9, 1.0)), lambda: KSAdamW([torch.nn.Parameter(torch.zeros(4, 6, device="cuda").t())])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(AssertionError):
        KSAdamW([torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=torch.float64))])


def params(prec, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(*shape, generator=g) * 0.1).to(DT[prec]).cuda()) for shape in ((5,), (64, 33), (1,), (128,), (7, 3, 2))]


def grads_of(ps, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(p.shape, generator=g).to(p.dtype).cuda() for p in ps]


def test_the_optimiser_against_torchs():
    """fp32: torch's AdamW in float64.  Ten steps, each off by 1e-6 of the change and the value at most."""
    from ksmm_amd import KSAdamW

    mine, theirs = params("fp32"), [torch.nn.Parameter(p.detach().double()) for p in params("fp32")]
    a, b = KSAdamW(mine, lr=1e-2, weight_decay=0.1), torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.1)
    for t in range(10):
        for p, q, g in zip(mine, theirs, grads_of(mine, t)):
            p.grad, q.grad = g, g.double()
        if t == 4:  # a parameter without a gradient is left as it is, and counts its own steps
            mine[1].grad = theirs[1].grad = None
        version = mine[0]._version
        a.step()
        b.step()
        assert mine[0]._version > version
    for p, q in zip(mine, theirs):
        assert float((p.double() - q).abs().max()) <= 10 * 1e-6 * 0.5


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("prec", ["fp32", "fp16"])
def test_state_goes_through_a_checkpoint(prec, bits, tmp_path):
    from ksmm_amd import KSAdamW

    ps, qs = params(prec), params(prec)
    a = KSAdamW(ps, bits=bits, seed=5)
    for t in range(3):
        for p, g in zip(ps, grads_of(ps, t)):
            p.grad = g
        a.step()
    torch.save({"w": [p.detach() for p in ps], "opt": a.state_dict()}, tmp_path / "c.pt")
    saved = torch.load(tmp_path / "c.pt", weights_only=True, map_location="cpu")
    b = KSAdamW(qs, bits=bits)
    b.load_state_dict(saved["opt"])
    for q, w in zip(qs, saved["w"]):
        q.data.copy_(w)
    for opt, which in ((a, ps), (b, qs)):
        for t in range(3, 6):
            for p, g in zip(which, grads_of(which, t)):
                p.grad = g
            opt.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        assert all(torch.equal(a.state[p][k], b.state[q][k]) and a.state[p][k].dtype == b.state[q][k].dtype for k in ("exp_avg", "exp_avg_sq"))


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_steps_count_on(bits):
    from ksmm_amd import KSAdamW

    ps, qs = params("fp16"), params("fp16")
    a, b = KSAdamW(ps, bits=bits, capturable=True), KSAdamW(qs, bits=bits)
    for which in (ps, qs):
        for p, g in zip(which, grads_of(which, 0)):
            p.grad = g.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for t in range(1, 5):
        for p, q, g in zip(ps, qs, grads_of(ps, t)):
            p.grad.copy_(g)
            q.grad.copy_(g)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        for p, q in zip(ps, qs):
            # the corrections are found in 64 bits on both sides and rounded once
            assert float((a.state[p]["master"] - b.state[q]["master"]).abs().max()) <= 1e-6
            if bits == 8:
                assert torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])


def test_beside_muon():
    """A block of 4-bit products: factors by KSMuon, the rest by KSAdamW, then served packed."""
    from ksmm_amd import KSAdamW, KSFeedForwardMX, KSMuon

    torch.manual_seed(0)
    block = KSFeedForwardMX((1, 128, 64, 2), [(1, 64, 128, 2)])
    muon, rest = KSMuon(block), KSAdamW(KSMuon.others(block), bits=8, grad_scale=1 / 64)
    x = torch.randn(50, 128, device="cuda").half()
    before = [p.detach().clone() for p in block.parameters()]
    for _ in range(3):
        with torch.enable_grad():
            n, r = block(block.begin(x), x)
            (n.float().square().mean() * 64).backward()
        muon.step()
        rest.step()
        block.zero_grad()
    assert all(not torch.equal(p, q) and torch.isfinite(p).all() for p, q in zip(block.parameters(), before))
    served = block.packed()
    assert torch.equal(served(block.begin(x), x)[0], block(block.begin(x), x)[0])


@pytest.mark.parametrize("bits", [8, 32])
def test_without_the_native_module(monkeypatch, bits):
    from ksmm_amd import _lib, adamw_moments, adamw_update

    def everything():
        s = make([100, 4097], "fp16", bits, True)
        adamw_update(s["w"], s["g"], s["m"], s["v"], s["scales"], s["master"], step=torch.full((1,), 9, device="cuda"), seed=4, **HOW)
        version = s["w"][0]._version
        adamw_update(s["w"], s["g"], s["m"], s["v"], s["scales"], s["master"], step=10, seed=4, **HOW)
        assert s["w"][0]._version > version
        out = s["w"] + s["m"] + s["v"] + s["master"]
        return out + (sum(map(list, adamw_moments(s["m"], s["v"], s["scales"])), []) if bits == 8 else [])

    native = everything()
    assert _lib.native() is not _lib._NoNative
    monkeypatch.setattr(_lib, "_native", _lib._NoNative)
    for x, y in zip(native, everything()):
        assert torch.equal(x, y)


def test_places_beyond_31_bits_of_bytes():
    """A tensor of almost 2^31 values: its ends as tensors of their own, rounded by the hash of their own places."""
    from ksmm_amd import adamw_moments, adamw_update

    n, k = (1 << 31) - 16384, 4096
    w = torch.zeros(n, dtype=torch.float16, device="cuda")
    g = torch.zeros(n, dtype=torch.float16, device="cuda")
    m, v, s = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(2, n // 32, dtype=torch.uint8, device="cuda")
    part = make([k], "fp16", 8, False)
    for at in (0, n - k):
        w[at:at + k], g[at:at + k], m[at:at + k], v[at:at + k] = part["w"][0], part["g"][0], part["m"][0], part["v"][0]
        s[:, at // 32:(at + k) // 32] = part["scales"][0]
    adamw_update([w], [g], [m], [v], [s], step=5, seed=2, **HOW)
    m0, v0 = R.decode_moments(part["m"][0], part["v"][0], part["scales"][0])
    w1, m1, v1 = R.adamw(part["w"][0].cpu().double(), part["g"][0], m0, v0, 5, HOW["lr"], HOW["betas"], HOW["eps"], HOW["weight_decay"], HOW["grad_scale"])
    key = R._mix((R._mix(2) + 5) & 0xFFFFFFFF)
    for at in (0, n - k):
        h = R._mix(torch.arange(at, at + k, dtype=torch.int64) ^ key)
        cm, cv, sc = R.encode_moments(m1, v1, (h & 0xFFFF).double() / 65536, (h >> 16).double() / 65536)
        assert torch.equal(s[:, at // 32:(at + k) // 32].cpu(), sc)
        got = R.decode_moments(m[at:at + k], v[at:at + k], s[:, at // 32:(at + k) // 32])
        assert all(torch.equal(x, y) for x, y in zip(got, R.decode_moments(cm, cv, sc)))
        assert float((w[at:at + k].cpu().double() - w1).abs().max()) <= 2.0 ** -11 * float(w1.abs().max()) + 1e-6
    assert not w[k:k + 1000].any() and not m[n // 2:n // 2 + 1000].any()


def test_threads_at_once():
    import threading

    from ksmm_amd import adamw_update

    alone, sets = [], []
    for i in range(4):
        s = make([1000 + i, 77], "fp32", 8, False, seed=i)
        adamw_update(s["w"], s["g"], s["m"], s["v"], s["scales"], seed=i, **HOW)
        alone.append(s)
        sets.append(make([1000 + i, 77], "fp32", 8, False, seed=i))
    torch.cuda.synchronize()

    def work(s, i):
        with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
            adamw_update(s["w"], s["g"], s["m"], s["v"], s["scales"], seed=i, **HOW)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(s, i)) for i, s in enumerate(sets)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for x, y in zip(alone, sets):
        assert all(torch.equal(p, q) for k in ("w", "m", "v", "scales") for p, q in zip(x[k], y[k]))


def test_captures_that_would_not_count_are_refused():
    from ksmm_amd import KSAdamW

    for how, before in ((dict(), 1), (dict(capturable=True), 0)):
        ps = params("fp16")
        opt = KSAdamW(ps, **how)
        for p, g in zip(ps, grads_of(ps, 0)):
            p.grad = g.clone()
        for _ in range(before):
            opt.step()
        kept = [p.detach().clone() for p in ps]
        with pytest.raises(RuntimeError, match="captur"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                opt.step()
        assert all(torch.equal(p, k) for p, k in zip(ps, kept))
