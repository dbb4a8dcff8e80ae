"""The training operators on the GPU -- norm and its gradients, balance loss,
gradient of the router logits, gradients of the router product -- against
plain implementations in 64 bits, and gradients against differences of these.

Tolerances count roundings.  u = 2^-24 is a rounding of fp32, h the rounding
of the output's type (2^-9 times the value for bf16, a half step of its eps /
2 = 2^-8 at most; fp32 u).  A sum over N values by threads that add at most 64
of them in turn, then 6 + 4 levels of a tree, is off by at most
(64 + 10) u times the sum of magnitudes; 128 u below covers it with the few
roundings of its terms."""
import ctypes

import pytest
import torch

from q36_amd import moe, synth

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    return torch.device("cuda:0")


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g)


def _within(got, ref, tol, what):
    got, tol = got.double().cpu(), tol.broadcast_to(ref.shape)
    bad = ~((got - ref).abs() <= tol)
    if bool(bad.any()):
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{what}{at}: {float(got[at])} for {float(ref[at])}, {float(tol[at]):.3g} allowed; {int(bad.sum())} values off")


# --------------------------------------------------------------------------
# norm
# --------------------------------------------------------------------------
def _norm_ref(v, w, b, rms, eps):
    """(y, n, r, d) in 64 bits of rows v."""
    d = v if rms else v - v.mean(1, keepdim=True)
    r = (d.square().mean(1, keepdim=True) + eps).rsqrt()
    n = d * r
    y = n if w is None else n * w
    return (y if b is None else y + b), n, r, d


def _wide(t, pad, dev, dtype, sentinel=False):
    """t on the GPU as the left part of wider rows."""
    T, D = t.shape
    buf = torch.full((T, D + pad), float("nan"), dtype=dtype, device=dev)
    buf[:, :D] = t.to(dev).to(dtype)
    return buf[:, :D]


NORM_SHAPES = [(1, 1), (4, 1), (3, 2), (1, 7), (5, 8), (2, 63), (9, 64), (1, 255), (4, 257), (3, 511), (5, 513), (7, 1023),
               (1, 2048), (61, 2048), (2, 2049), (3, 4095), (2, 4097), (2, 8191), (3, 8192), (2, 8193), (2, 16383),
               (1, 16384), (1030, 130)]


@pytest.mark.parametrize("T,D", NORM_SHAPES)
@pytest.mark.parametrize("xt,yt,rms,add,pad", [(F32, F32, False, False, 0), (F32, BF16, True, True, 3),
                                              (BF16, BF16, False, True, 1), (BF16, F32, True, False, 0)])
def test_layernorm(dev, T, D, xt, yt, rms, add, pad):
    g = _g(T * 20000 + D)
    x = _wide(_randn(g, T, D) * 2 + 0.5, pad, dev, xt)
    a = _wide(_randn(g, T, D), pad, dev, xt) if add else None
    w = 1 + 0.2 * _randn(g, D) if D % 3 else None
    b = 0.1 * _randn(g, D) if not rms and D % 2 else None
    eps = 1e-6
    y, h = moe.layernorm(x, None if w is None else w.to(dev), None if b is None else b.to(dev), a=a, eps=eps, rms=rms,
                         out_dtype=yt)
    assert y.dtype == yt and (h is None) == (not add)
    v = x.double().cpu() + (a.double().cpu() if add else 0)
    ref, n, r, d = _norm_ref(v, None if w is None else w.double(), None if b is None else b.double(), rms, eps)
    if add:
        _within(h, v, HALF[xt] * v.abs() + U * v.abs(), "h")
    ww = torch.ones(D).double() if w is None else w.double().abs()
    # d is off by the mean's error (128 u of the mean |d|) and, of a sum, by the
    # sum's rounding; r by half the squares' 128 u and 2 u of its own
    off = U * (128 * d.abs().mean(1, keepdim=True) + 2 * d.abs() + (4 * v.abs() if add else 0)) * r * ww \
        + U * (96 + 128) * (n * ww).abs() + 2 * U * ref.abs()
    _within(y, ref, off + HALF[yt] * ref.abs(), "y")


@pytest.mark.parametrize("D", [100, 2048, 5000])
def test_layernorm_far_offset_and_outliers(dev, D):
    """Rows whose offset is 10^4 times their spread, and rows with one value
    10^4 times the others: what one pass over squares would lose."""
    g = _g(D)
    x = _randn(g, 4, D)
    x[0] += 1e4
    x[1] -= 3e4
    x[2, D // 2] = 1e4
    x[3] *= 1e-12
    x = x.to(dev)
    y, _ = moe.layernorm(x, eps=1e-6)
    v = x.double().cpu()
    ref, n, r, d = _norm_ref(v, None, None, False, 1e-6)
    # the first mean may be off by 128 u |mean|, which makes the deviations that
    # much larger, and their roundings with them
    big = d.abs() + 128 * U * v.abs()
    off = U * r * (128 * big.mean(1, keepdim=True) + 2 * big) + U * 256 * n.abs() * (big.square().mean(1, keepdim=True).sqrt() * r)
    _within(y, ref, off + U * ref.abs(), "y")


def test_layernorm_constant_and_zero_rows(dev):
    x = torch.stack([torch.full((300,), 3.0), torch.zeros(300), torch.full((300,), -1e30)]).to(dev)
    b = torch.arange(300.0).to(dev)
    y, _ = moe.layernorm(x, None, b, eps=1e-6)
    # 300 equal powers of the sum round: the deviation that is left times 1/sqrt(eps)
    assert torch.equal(y[1], b)
    assert float((y[0] - b).abs().max()) <= 3.0 * 4 * U * 1e3 + 300 * U
    z, _ = moe.layernorm(x[:2], rms=True, eps=1e-6)
    assert torch.equal(z[1], torch.zeros_like(z[1])) and float((z[0] - 1).abs().max()) <= 1e-6


@pytest.mark.parametrize("rms", [False, True])
def test_layernorm_keeps_nan_and_inf_in_their_rows(dev, rms):
    x = _randn(_g(4), 6, 777).to(dev)
    clean, _ = moe.layernorm(x, rms=rms)
    x2 = x.clone()
    x2[1, 5], x2[3, 776], x2[4, 0] = float("nan"), float("inf"), -float("inf")
    y, _ = moe.layernorm(x2, rms=rms)
    for t in (0, 2, 5):
        assert torch.equal(y[t], clean[t])
    assert bool(y[1].isnan().all()) and bool(y[3].isnan().any()) and bool(y[4].isnan().any())


def test_layernorm_in_place_sum_and_untouched_surroundings(dev):
    """h written over x, and over a; the columns between rows and the rows
    after the last one keep what they held."""
    L = moe.lib()
    T, D, ld = 5, 1001, 1010
    g = _g(8)
    for xt, fmt in ((F32, 0), (BF16, 1)):
        x0 = _randn(g, T + 2, ld).to(dev).to(xt)
        a0 = _randn(g, T + 2, ld).to(dev).to(xt)
        want_y, want_h = moe.layernorm(x0[:T, :D], a=a0[:T, :D], out_dtype=F32)
        for over in ("x", "a"):
            x, a = x0.clone(), a0.clone()
            y = torch.full((T + 2, ld), 7.0, device=dev)
            h = x if over == "x" else a
            rc = L.q36moe_layernorm(x.data_ptr(), ld, a.data_ptr(), ld, fmt, None, None, T, D, ctypes.c_float(1e-6), 0,
                                    h.data_ptr(), ld, y.data_ptr(), ld, 0, moe._stream())
            torch.cuda.synchronize()
            assert rc == 0
            assert torch.equal(y[:T, :D], want_y) and torch.equal(h[:T, :D], want_h)
            assert bool((y[:T, D:] == 7).all()) and bool((y[T:] == 7).all())
            old = x0 if over == "x" else a0
            assert torch.equal(h[:, D:], old[:, D:]) and torch.equal(h[T:], old[T:])


def _norm_grad_ref(dy, v, w, rms, eps):
    _, n, r, d = _norm_ref(v, None, None, rms, eps)
    gw = dy if w is None else dy * w
    core = gw - n * (gw * n).mean(1, keepdim=True)
    if not rms:
        core = core - gw.mean(1, keepdim=True)
    return core * r, (dy * n).sum(0), dy.sum(0), n, r, gw


@pytest.mark.parametrize("T,D", NORM_SHAPES + [(513, 600), (1500, 2048), (2000, 40)])
@pytest.mark.parametrize("xt,yt,rms,add,pad", [(F32, F32, True, True, 0), (F32, BF16, False, False, 3),
                                              (BF16, BF16, False, True, 1), (BF16, F32, True, False, 0)])
def test_layernorm_backward(dev, T, D, xt, yt, rms, add, pad):
    g = _g(T * 20000 + D + 1)
    h = _wide(_randn(g, T, D) * 2 + 0.5, pad, dev, xt)
    dy = _wide(_randn(g, T, D), pad, dev, yt)
    dres = _wide(_randn(g, T, D), pad, dev, xt) if add else None
    w = 1 + 0.2 * _randn(g, D) if D % 3 else None
    eps = 1e-6
    dx, dw, db = moe.layernorm_backward(dy, h, None if w is None else w.to(dev), dres=dres, eps=eps, rms=rms)
    assert (db is None) == rms and dx.dtype == xt
    dy64, res = dy.double().cpu(), dres.double().cpu() if add else 0
    rdx, rdw, rdb, n, r, gw = _norm_grad_ref(dy64, h.double().cpu(), None if w is None else w.double(), rms, eps)
    # n is off by 128 u of its mean magnitude and 256 u of itself; the row's sums
    # by 128 u of their terms' magnitudes
    dn = U * (128 * n.abs().mean(1, keepdim=True) + 256 * n.abs())
    mgn, mg = (gw * n).abs().mean(1, keepdim=True), gw.abs().mean(1, keepdim=True)
    emgn = 128 * U * mgn + (gw.abs() * dn).mean(1, keepdim=True)
    off = r * (8 * U * gw.abs() + 128 * U * mg + dn * mgn + n.abs() * emgn + 4 * U * n.abs() * mgn)
    off = off + 256 * U * rdx.abs()
    ref = rdx + res
    _within(dx, ref, off + U * ref.abs() + HALF[xt] * ref.abs(), "dx")
    # a stream adds its tokens in turn, 512 streams are added by 16 groups
    turns = T / 512 + 32 + 16 + 4
    _within(dw, rdw, (dy64.abs() * dn).sum(0) + turns * U * (dy64 * n).abs().sum(0), "dw")
    if db is not None:
        _within(db, rdb, turns * U * dy64.abs().sum(0), "db")


@pytest.mark.parametrize("rms", [False, True])
def test_layernorm_backward_against_differences(dev, rms):
    """Along random directions, the difference quotient of <dy, y> in 64 bits."""
    g = _g(31)
    T, D, eps = 5, 203, 1e-6
    h, dy, w, b = _randn(g, T, D), _randn(g, T, D), 1 + 0.2 * _randn(g, D), _randn(g, D)
    dx, dw, db = moe.layernorm_backward(dy.to(dev), h.to(dev), w.to(dev), eps=eps, rms=rms, want_db=True)

    def f(h, w, b):
        return float((_norm_ref(h, w, b, rms, eps)[0] * dy.double()).sum())

    h, w, b = h.double(), w.double(), b.double()
    for i in range(4):
        s = 1e-5
        vh, vw, vb = (_randn(g, *t.shape).double() for t in (h, w, b))
        quot = (f(h + s * vh, w + s * vw, b + s * vb) - f(h - s * vh, w - s * vw, b - s * vb)) / (2 * s)
        terms = [(dx.double().cpu() * vh), (dw.double().cpu() * vw), (db.double().cpu() * vb)]
        # the quotient's own error is of order s^2 of third derivatives and
        # 2^-53 |f| / s, both under 1e-8; 256 u of the terms is the kernel's
        size = sum(float(t.abs().sum()) for t in terms)
        assert abs(sum(float(t.sum()) for t in terms) - quot) <= (256 * U + 1e-8) * size


def test_layernorm_backward_wants(dev):
    """Every subset of the outputs has the same bits; no tokens clear the sums."""
    g = _g(3)
    h, dy, w = _randn(g, 70, 300).to(dev), _randn(g, 70, 300).to(dev), _randn(g, 300).to(dev)
    full = moe.layernorm_backward(dy, h, w)
    for wx in (True, False):
        for ww in (True, False):
            for wb in (True, False):
                if not (wx or ww or wb):
                    continue
                got = moe.layernorm_backward(dy, h, w, want_dx=wx, want_dw=ww, want_db=wb)
                for o, f, on in zip(got, full, (wx, ww, wb)):
                    assert (o is None) != on and (o is None or torch.equal(o, f))
    dx, dw, db = moe.layernorm_backward(dy[:0], h[:0], w)
    assert dx.shape == (0, 300) and float(dw.abs().sum()) == 0.0 and float(db.abs().sum()) == 0.0
    with pytest.raises(moe.Q36MoEError):
        moe.layernorm_backward(dy, h, w, want_dx=False, want_dw=False, want_db=False)


def test_layernorm_matches_the_quantising_producer(dev):
    """The framework's add + RMSNorm computes the same rows."""
    g = _g(5)
    h0, a, w = _randn(g, 33, 2048).to(dev), _randn(g, 33, 2048).to(dev), (1 + 0.1 * _randn(g, 2048)).to(dev)
    h = h0.clone()
    y, _, _ = moe.add_rmsnorm_quant(h, a, w, eps=1e-6, want_q=False)
    y2, h2 = moe.layernorm(h0, w, a=a, eps=1e-6, rms=True)
    assert torch.equal(h, h2)
    # sums of squares in two orders: 2 x 64 u of the mean, half of that in the root
    assert float(((y - y2).abs() / y.abs().clamp_min(1e-30)).max()) <= 70 * U


# --------------------------------------------------------------------------
# balance loss and gradient of the logits
# --------------------------------------------------------------------------
def _probs(l):
    m = l.amax(1, keepdim=True)
    m = torch.where(m == -float("inf"), torch.zeros_like(m), m)
    e = (l - m).exp()
    s = e.sum(1, keepdim=True)
    return torch.where(s > 0, e / s, torch.zeros_like(e))


def _balance_ref(l, idx, live, k, coef):
    E = l.shape[1]
    p = _probs(l)[live]
    psum = p.sum(0)
    flat = idx[live].reshape(-1)
    flat = flat[(flat >= 0) & (flat < E)].long()
    counts = torch.bincount(flat, minlength=E)
    n = int(live.sum())
    loss = coef * E / (k * n * n) * float((counts.double() * psum).sum()) if n else 0.0
    return loss, counts, n, psum


def _routing(g, T, E, k, spread=1.0):
    l = spread * _randn(g, T, E)
    return l, torch.sort(l, dim=1, descending=True, stable=True).indices[:, :k].int()


def _live(g, T, mask):
    if mask == "none":
        return None, torch.ones(T, dtype=torch.bool)
    m = torch.rand(T, generator=g) < 0.7
    if mask == "dead":
        m[:] = False
    return m, m


# |x| of exp(x) costs no more than its own rounding (x - max: u |x|) and 3 u
def _p_err(l):
    m = torch.where(l.isfinite(), l, torch.zeros_like(l)).double()
    return U * (2 * (m.amax(1, keepdim=True) - m.amin(1, keepdim=True)) + 40)


ROUTE_SHAPES = [(1, 1, 1), (1, 8, 8), (2, 3, 2), (15, 17, 1), (16, 16, 3), (17, 60, 4), (64, 64, 8), (61, 65, 5),
                (203, 256, 8), (256, 255, 7), (257, 256, 8), (384, 100, 2), (385, 256, 8), (390, 1, 1),
                (1000, 129, 6), (16500, 256, 8)]


@pytest.mark.parametrize("T,E,k", ROUTE_SHAPES)
@pytest.mark.parametrize("mask", ["none", "some", "dead"])
def test_balance_loss(dev, T, E, k, mask):
    g = _g(T * 1000 + E)
    l, idx = _routing(g, T, E, k, 3.0)
    m, live = _live(g, T, mask)
    ld = l.to(dev)
    if m is not None:
        ld = ld.clone()
        ld[~m.to(dev)] = float("nan")      # padding holds anything
    loss, counts, psum = moe.balance_loss(ld, idx.to(dev), coef=0.3, mask=None if m is None else m.to(dev))
    rl, rc, n, rp = _balance_ref(l.double(), idx, live, k, 0.3)
    assert torch.equal(counts.cpu(), torch.cat([rc, torch.tensor([n])]).int())
    # tokens per thread of a workgroup, its 16 waves, and up to 128 workgroups
    turns = T / 64 / min(128, max(1, T / 128)) + 16 + 32 + 8
    err = float(_p_err(l).max()) + turns * U
    _within(psum, rp, err * rp, "psum")
    assert abs(float(loss) - rl) <= (err + 2 * U) * rl


def test_balance_loss_perfect_balance_is_coef(dev):
    """Equal logits and picks spread evenly: the loss is coef."""
    E, k, T = 32, 4, 64
    idx = (torch.arange(T * k) % E).view(T, k).int().to(dev)
    loss, counts, _ = moe.balance_loss(torch.full((T, E), 2.5, device=dev), idx, coef=0.125)
    assert counts[:E].eq(T * k // E).all() and abs(float(loss) - 0.125) <= 0.125 * 8 * U


def test_balance_loss_dropped_picks_ld_and_infinities(dev):
    """Indices that name no expert are not counted, experts switched off by
    -inf have no share, a token with nothing but -inf none at all; the columns
    past n_expert are not read."""
    g = _g(17)
    T, E, k = 300, 40, 4
    l, idx = _routing(g, T, E, k)
    l[:, 3] = -float("inf")
    l[5] = -float("inf")
    l[6] = torch.finfo(F32).min            # all of one value: 1/E each
    l[7, 1:] = torch.finfo(F32).min        # all on one expert
    idx[::7, 2], idx[::11, 0] = -1, E
    idx[9] = 12                            # one expert four times
    buf = torch.full((T, E + 9), float("nan"))
    buf[:, :E] = l
    loss, counts, psum = moe.balance_loss(buf.to(dev), idx.to(dev), n_expert=E)
    rl, rc, n, rp = _balance_ref(l.double(), idx, torch.ones(T, dtype=torch.bool), k, 1.0)
    assert torch.equal(counts.cpu(), torch.cat([rc, torch.tensor([n])]).int())
    _within(psum, rp, 200 * U * rp, "psum")
    assert abs(float(loss) - rl) <= 200 * U * rl and float(psum[3]) <= 1.0 / E + 1e-6


def test_balance_loss_without_tokens(dev):
    loss, counts, psum = moe.balance_loss(torch.zeros((0, 20), device=dev), torch.zeros((0, 2), dtype=torch.int32, device=dev))
    assert float(loss) == 0.0 and not bool(counts.any()) and not bool(psum.any())


def _logit_grad_ref(l, idx, dwt, scale, renorm, counts, coef, dloss, live, k):
    T, E = l.shape
    p, out, mag = _probs(l), torch.zeros_like(l), torch.zeros_like(l)
    ok = (idx >= 0) & (idx < E)
    at = idx.clamp(0, E - 1).long()
    if dwt is not None:
        up = torch.where(ok, dwt * scale, torch.zeros_like(dwt))
        if renorm:
            q = _probs(torch.where(ok, l.gather(1, at), torch.full_like(up, -float("inf"))))
            s = q * (up - (q * up).sum(1, keepdim=True))
            out.scatter_add_(1, at, torch.where(ok, s, torch.zeros_like(s)))
            mag.scatter_add_(1, at, q * (up.abs() + (q * up).abs().sum(1, keepdim=True)))
        else:
            u, ua = torch.zeros_like(l).scatter_add_(1, at, up), torch.zeros_like(l).scatter_add_(1, at, up.abs())
            out += p * (u - (p * u).sum(1, keepdim=True))
            mag += p * (ua + (p * ua).sum(1, keepdim=True))
    if counts is not None:
        n = counts[E].double()
        if n > 0:
            f = counts[:E].double() / (n * k)
            gain = dloss * coef * E / n
            out += gain * p * (f - (p * f).sum(1, keepdim=True))
            mag += gain.abs() * p * (f + (p * f).sum(1, keepdim=True))
    return out * live[:, None], mag


@pytest.mark.parametrize("T,E,k", ROUTE_SHAPES)
@pytest.mark.parametrize("parts,renorm,mask", [("both", True, "some"), ("both", False, "none"), ("weights", True, "none"),
                                               ("weights", False, "some"), ("balance", True, "none"), ("both", True, "dead")])
def test_router_topk_backward(dev, T, E, k, parts, renorm, mask):
    g = _g(T * 1000 + E + 7)
    l, idx = _routing(g, T, E, k, 2.0)
    m, live = _live(g, T, mask)
    dwt = _randn(g, T, k) if parts != "balance" else None
    counts = dloss = None
    if parts != "weights":
        rc = _balance_ref(l.double(), idx, live, k, 1.0)
        counts = torch.cat([rc[1], torch.tensor([rc[2]])]).int()
        dloss = torch.tensor(1.7)
    buf = torch.full((T, E + 3), float("nan"))
    buf[:, :E] = l
    up = dwt
    if m is not None:
        buf[~m] = float("inf")
        if dwt is not None:
            up = dwt.clone()
            up[~m] = float("nan")
    to = lambda t: None if t is None else t.to(dev)
    got = moe.router_topk_backward(buf.to(dev), to(idx), to(up), scale=1.25, renorm=renorm, counts=to(counts), coef=0.7,
                                   mask=to(m), dloss=to(dloss), n_expert=E)
    ref, mag = _logit_grad_ref(l.double(), idx, None if dwt is None else dwt.double(), 1.25, renorm, counts, 0.7,
                               None if dloss is None else dloss.double(), live, k)
    # two factors p, each as exact as _p_err says, and sums of 16 values per lane
    _within(got, ref, (3 * _p_err(l) + 40 * U) * mag, "dlogits")
    if m is not None:
        assert not bool(got[~m.to(dev)].any())


def test_router_topk_backward_odd_picks(dev):
    """An expert picked twice gets both gradients, a dropped pick none, experts
    at -inf none; a token whose picks are all at -inf or all dropped has no
    gradient."""
    g = _g(23)
    T, E, k = 40, 50, 6
    l, idx = _routing(g, T, E, k)
    idx[3] = 11
    idx[4, 1] = idx[4, 4]
    idx[5, 2], idx[6, 0] = -1, E + 100
    idx[7] = -1
    l[8, idx[8, 2].long()] = -float("inf")
    l[9, idx[9].long()] = -float("inf")
    l[10] = -float("inf")
    l[11, idx[11].long()] = torch.finfo(F32).min
    dwt = _randn(g, T, k)
    counts = torch.randint(0, 20, (E + 1,), generator=g).int()
    counts[E] = T
    for renorm in (True, False):
        for c in (None, counts):
            got = moe.router_topk_backward(l.to(dev), idx.to(dev), dwt.to(dev), renorm=renorm,
                                           counts=None if c is None else c.to(dev), coef=0.5)
            ref, mag = _logit_grad_ref(l.double(), idx, dwt.double(), 1.0, renorm, c, 0.5, torch.tensor(1.0).double(),
                                       torch.ones(T, dtype=torch.bool), k)
            assert bool(got.isfinite().all())
            # row 11's spread is the type's whole range, where p is 0 or its picks' share
            lim = 300 * U * mag
            _within(got, ref, lim, "dlogits")


@pytest.mark.parametrize("renorm", [True, False])
def test_router_topk_backward_against_differences(dev, renorm):
    g = _g(29)
    T, E, k, coef, scale = 9, 33, 5, 0.4, 1.5
    l, idx = _routing(g, T, E, k)
    dwt = _randn(g, T, k)
    loss, counts, _ = moe.balance_loss(l.to(dev), idx.to(dev), coef=coef)
    got = moe.router_topk_backward(l.to(dev), idx.to(dev), dwt.to(dev), scale=scale, renorm=renorm, counts=counts,
                                   coef=coef).double().cpu()

    def f(l):
        wt = _probs(l).gather(1, idx.long())
        if renorm:
            wt = wt / wt.sum(1, keepdim=True)
        return float((scale * wt * dwt.double()).sum()) + _balance_ref(l, idx, torch.ones(T, dtype=torch.bool), k, coef)[0]

    l = l.double()
    assert abs(float(loss) - _balance_ref(l, idx, torch.ones(T, dtype=torch.bool), k, coef)[0]) <= 1e-5 * coef
    for i in range(4):
        v, s = _randn(g, T, E).double(), 1e-5
        quot = (f(l + s * v) - f(l - s * v)) / (2 * s)
        assert abs(float((got * v).sum()) - quot) <= (200 * U + 1e-8) * float((got * v).abs().sum())


def test_router_topk_backward_strided_rows_keep_their_surroundings(dev):
    L = moe.lib()
    g = _g(41)
    T, E, k, ld = 21, 37, 3, 44
    l, idx = _routing(g, T, E, k)
    dwt = _randn(g, T, k).to(dev)
    out = torch.full((T + 2, ld), 7.0, device=dev)
    want = moe.router_topk_backward(l.to(dev), idx.to(dev), dwt)
    ld_, id_ = l.to(dev), idx.to(dev)
    rc = L.q36moe_router_topk_backward(ld_.data_ptr(), E, id_.data_ptr(), dwt.data_ptr(), None, None, None, T, E, k,
                                       ctypes.c_float(1), 1, ctypes.c_float(1), out.data_ptr(), ld, moe._stream())
    torch.cuda.synchronize()
    assert rc == 0 and torch.equal(out[:T, :E], want) and bool((out[:T, E:] == 7).all()) and bool((out[T:] == 7).all())


# --------------------------------------------------------------------------
# gradients of the router product
# --------------------------------------------------------------------------
@pytest.mark.parametrize("T,E,shared", [(1, 1, False), (1, 256, True), (2, 7, True), (17, 256, True), (31, 33, False),
                                        (33, 8, True), (64, 255, False), (100, 32, True), (203, 256, True), (257, 257, True),
                                        (300, 300, False), (513, 256, False), (700, 60, True), (1025, 256, True),
                                        (1100, 600, True), (2500, 128, True), (4097, 256, True), (640, 256, True), (641, 131, False),
                                        (1025, 65, True), (1401, 20, True), (3001, 7, False)])
@pytest.mark.parametrize("xt", [F32, BF16])
def test_router_logits_backward(dev, T, E, shared, xt):
    g = _g(T * 1000 + E)
    rows = E + shared
    w = (_randn(g, rows, 2048) * 0.02)
    x = _randn(g, T, 2048).to(xt)
    # gradients of very different sizes in one row, as a softmax leaves them
    d = _randn(g, T, rows) * torch.exp(3 * _randn(g, T, rows))
    buf = torch.full((T, E + 2 + shared), float("nan"))
    buf[:, :E] = d[:, :E]
    if shared:
        buf[:, -1] = d[:, E]
    buf = buf.to(dev)
    dw, dx = moe.router_logits_backward(w.to(dev), x.to(dev), E, buf[:, :E], buf[:, -1] if shared else None)
    d64, x64, w64 = d.double(), x.double(), w.double()
    # fp32 sums of N products: N roundings, each at most u times a partial sum
    # and so u times the sum of magnitudes (one large term keeps every later
    # partial sum that large).  Uniform in +-u they have a deviation of u / sqrt(3),
    # N of them sqrt(N / 3) u, and six deviations are not reached in the 10^7
    # values here (10^-9 each); 8 u for the products and the sum's last levels.
    mag_w, mag_x = d64.abs().T @ x64.abs(), d64.abs() @ w64.abs()
    ref_w, ref_x = d64.T @ x64, d64 @ w64
    few = lambda n: (8 + 6 * (n / 3) ** 0.5) * U
    _within(dw, ref_w, few(T) * mag_w, "dw")
    # a bf16 result may be formed from operands of 16 bits
    lost = few(rows) + (0 if xt == F32 else 2.0 ** -14)
    _within(dx, ref_x, lost * mag_x + HALF[xt] * ref_x.abs(), "dx")


@pytest.mark.parametrize("T", [50, 1500])
def test_router_logits_backward_wants_and_empty(dev, T):
    g = _g(2)
    w, x, d = _randn(g, 20, 2048).to(dev), _randn(g, T, 2048).to(dev), _randn(g, T, 20).to(dev)
    dw, dx = moe.router_logits_backward(w, x, 20, d)
    a, b = moe.router_logits_backward(w, x, 20, d, want_dw=False)
    assert a is None and torch.equal(b, dx)
    a, b = moe.router_logits_backward(w, x, 20, d, want_dx=False)
    assert b is None and torch.equal(a, dw)
    dw, dx = moe.router_logits_backward(w, x[:0], 20, d[:0])
    assert dx.shape == (0, 2048) and not bool(dw.any())
    w, x = torch.zeros(257, 2048, device=dev), torch.zeros(0, 2048, device=dev)
    dw, _ = moe.router_logits_backward(w, x, 256, torch.zeros(0, 256, device=dev), torch.zeros(0, device=dev))
    assert dw.shape == (257, 2048) and not bool(dw.any())
    with pytest.raises(moe.Q36MoEError):
        moe.router_logits_backward(w, x, 19, d[:, :19])          # a row of the shared gate without its gradient
    with pytest.raises(moe.Q36MoEError):
        moe.router_logits_backward(w, x, 20, d[:, :19])


@pytest.mark.parametrize("T", [40, 2000])
def test_router_logits_backward_zero_gradients_and_infinities(dev, T):
    """Zero gradients give exact zeros; a value that is not finite reaches the
    results it enters, and none of the others."""
    g = _g(T)
    w, x = (_randn(g, 257, 2048) * 0.02).to(dev), _randn(g, T, 2048).to(dev)
    z = torch.zeros(T, 256, device=dev)
    dw, dx = moe.router_logits_backward(w, x, 256, z, z[:, 0])
    assert not bool(dw.any()) and not bool(dx.any())
    d = _randn(g, T, 256).to(dev)
    s = _randn(g, T).to(dev)
    dw0, dx0 = moe.router_logits_backward(w, x, 256, d, s)
    d[7, 100] = float("inf")
    dw1, dx1 = moe.router_logits_backward(w, x, 256, d, s)
    assert not bool(dw1[100].isfinite().any()) and not bool(dx1[7].isfinite().any())
    keep_r, keep_t = torch.arange(257, device=dev) != 100, torch.arange(T, device=dev) != 7
    assert torch.equal(dw1[keep_r], dw0[keep_r]) and torch.equal(dx1[keep_t], dx0[keep_t])


@pytest.mark.parametrize("xt", [F32, BF16])
def test_router_logits_backward_growing_values(dev, xt):
    """Values that grow along the tokens by factors of 10^4 at places of their
    own per row and column (and rows and columns that begin with zeros, or are
    zero throughout): the sums before and after a jump keep fp32's exactness."""
    T, E = 2600, 256
    g = _g(91)
    d, x, w = _randn(g, T, E + 1), _randn(g, T, 2048), 0.02 * _randn(g, E + 1, 2048)
    at_d, at_x = torch.randint(0, T, (E + 1,), generator=g), torch.randint(0, T, (2048,), generator=g)
    tok = torch.arange(T)[:, None]
    d = torch.where(tok >= at_d, d * 1e4, d * (torch.arange(E + 1) % 5 != 2))
    x = torch.where(tok >= at_x, x * 1e4, x * (torch.arange(2048) % 7 != 3))
    d[:, 17], x[:, 100] = 0.0, 0.0
    d[:, 18] *= 1e-30
    x[:, 101] *= 1e-30
    x = x.to(xt)
    dw, dx = moe.router_logits_backward(w.to(dev), x.to(dev), E, d[:, :E].contiguous().to(dev), d[:, E].to(dev))
    d64, x64, w64 = d.double(), x.double(), w.double()
    few = lambda n: (8 + 6 * (n / 3) ** 0.5) * U
    # the product of the two small ones, 10^-51, is under fp32's range, whose
    # rounding there is 2^-150
    _within(dw, d64.T @ x64, few(T) * (d64.abs().T @ x64.abs()) + 2.0 ** -150, "dw")
    ref = d64 @ w64
    lost = few(E + 1) + (0 if xt == F32 else 2.0 ** -14)
    _within(dx, ref, lost * (d64.abs() @ w64.abs()) + HALF[xt] * ref.abs(), "dx")


# --------------------------------------------------------------------------
# all of them
# --------------------------------------------------------------------------
def _calls(dev, seed, T=700, E=256, k=8):
    """One call of each operator on inputs of the seed."""
    g = _g(seed)
    x, a, dy = (_randn(g, T, 2048).to(dev) for _ in range(3))
    w, b = (1 + 0.1 * _randn(g, 2048)).to(dev), _randn(g, 2048).to(dev)
    l, idx = _routing(g, T, E, k)
    l, idx, dwt = l.to(dev), idx.to(dev), _randn(g, T, k).to(dev)
    mask = (torch.rand(T, generator=g) < 0.9).to(dev)
    rw, d, s = (0.02 * _randn(g, E + 1, 2048)).to(dev), _randn(g, T, E).to(dev), _randn(g, T).to(dev)

    def calls():
        loss, counts, psum = moe.balance_loss(l, idx, mask=mask)
        return [*moe.layernorm(x, w, b, a=a), *moe.layernorm_backward(dy, x, w, dres=a), loss, counts, psum,
                moe.router_topk_backward(l, idx, dwt, counts=counts, mask=mask),
                *moe.router_logits_backward(rw, x, E, d, s), *moe.router_logits_backward(rw, x.to(BF16), E, d, s)]
    return calls


@pytest.mark.parametrize("T", [1, 30, 700])
def test_same_bits_again_on_another_stream_and_in_a_graph(dev, T):
    calls, other = _calls(dev, 1, T), _calls(dev, 2, T)
    ref = [t.clone() for t in calls()]
    for t, r in zip(calls(), ref):
        assert torch.equal(t, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        here = calls()
        there = other()
    torch.cuda.synchronize()
    for t, r in zip(here, ref):
        assert torch.equal(t, r)
    graphs = []
    for c in (calls, other):          # two graphs in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = c()
        graphs.append((graph, outs, [t.clone() for t in (ref if c is calls else there)]))
    for _ in range(3):
        for graph, outs, want in graphs:
            for t in outs:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for t, r in zip(outs, want):
                assert torch.equal(t, r)
            for t, r in zip(calls(), ref):     # eager work between the replays
                assert torch.equal(t, r)


def test_two_streams_at_once(dev):
    a, b = _calls(dev, 5, 900), _calls(dev, 6, 1300)
    ra, rb = [t.clone() for t in a()], [t.clone() for t in b()]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            oa = a()
        with torch.cuda.stream(s2):
            ob = b()
        torch.cuda.synchronize()
        for t, r in zip(oa + ob, ra + rb):
            assert torch.equal(t, r)


def test_offsets_past_32_bits(dev):
    """Rows so far apart that their offsets need more than 32 bits, in elements
    and in bytes, give what the same rows give side by side."""
    g = _g(61)

    def far(rows, gap, dtype):
        T, n = rows.shape
        buf = torch.empty((T - 1) * gap + n, dtype=dtype, device=dev).as_strided((T, n), (gap, 1))
        return buf.copy_(rows.to(dev))

    x, dy = _randn(g, 4, 700).to(BF16), _randn(g, 4, 700)
    xf, gf = far(x, 2 ** 30 + 12, BF16), far(dy, 2 ** 29 + 4, F32)
    x, dy = x.to(dev), dy.to(dev)
    for a, b in ((moe.layernorm(xf, a=xf)[0], moe.layernorm(x, a=x)[0]),
                 *zip(moe.layernorm_backward(gf, xf, dres=xf), moe.layernorm_backward(dy, x, dres=x))):
        assert torch.equal(a, b)
    del xf, gf
    l, idx = _routing(g, 6, 130, 4)
    lf, idx, dwt = far(l, 2 ** 29 + 4, F32), idx.to(dev), _randn(g, 6, 4).to(dev)
    l = l.to(dev)
    got, want = moe.balance_loss(lf, idx), moe.balance_loss(l, idx)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(moe.router_topk_backward(lf, idx, dwt, counts=want[1]), moe.router_topk_backward(l, idx, dwt, counts=want[1]))
    del lf
    for T in (600, 700):
        w, x, d = (0.02 * _randn(g, 200, 2048)).to(dev), _randn(g, T, 2048).to(dev), _randn(g, T, 200)
        df = far(d, 2 ** 22, F32)
        for a, b in zip(moe.router_logits_backward(w, x, 200, df), moe.router_logits_backward(w, x, 200, d.to(dev))):
            assert torch.equal(a, b)
        del df


def test_python_refusals(dev):
    x = torch.zeros(4, 64, device=dev)
    idx = torch.zeros(4, 3, dtype=torch.int32, device=dev)
    bad = [lambda: moe.layernorm(x.half()), lambda: moe.layernorm(x[0]), lambda: moe.layernorm(x.T),
           lambda: moe.layernorm(x, torch.ones(63, device=dev)), lambda: moe.layernorm(x, torch.ones(64)),
           lambda: moe.layernorm(x, a=x[:3]), lambda: moe.layernorm(x, a=x.to(BF16)), lambda: moe.layernorm(x[:1].expand(4, 64)),
           lambda: moe.layernorm(x, out_dtype=torch.float16), lambda: moe.layernorm(x, eps=-1.0),
           lambda: moe.layernorm(torch.zeros(2, 0, device=dev)), lambda: moe.layernorm(torch.zeros(2, 16385, device=dev)),
           lambda: moe.layernorm_backward(x[:2], x), lambda: moe.layernorm_backward(x, x, dres=x.to(BF16)),
           lambda: moe.layernorm_backward(x.cpu(), x),
           lambda: moe.balance_loss(x.double(), idx), lambda: moe.balance_loss(x, idx.long()), lambda: moe.balance_loss(x, idx[:3]),
           lambda: moe.balance_loss(x, idx, mask=torch.ones(3, dtype=torch.bool, device=dev)),
           lambda: moe.balance_loss(x, idx, n_expert=65), lambda: moe.balance_loss(x[:, :40], idx, n_expert=45),
           lambda: moe.balance_loss(x, idx, n_expert=0), lambda: moe.balance_loss(x, idx, n_expert=-2),
           lambda: moe.router_topk_backward(x[:, :40], idx, x[:, :3].contiguous(), n_expert=45),
           lambda: moe.balance_loss(torch.zeros(4, 257, device=dev), idx),
           lambda: moe.balance_loss(x, torch.zeros(4, 9, dtype=torch.int32, device=dev)),
           lambda: moe.balance_loss(x, torch.zeros(4, 6, dtype=torch.int32, device=dev)[:, ::2]),
           lambda: moe.router_topk_backward(x, idx), lambda: moe.router_topk_backward(x, idx, x[:, :2]),
           lambda: moe.router_topk_backward(x, idx, counts=torch.zeros(64, dtype=torch.int32, device=dev)),
           lambda: moe.router_topk_backward(x, idx, x[:, :3].contiguous(), dloss=torch.zeros(2, device=dev)),
           lambda: moe.router_logits_backward(x, x, 4, x[:, :4])]
    for i, call in enumerate(bad):
        with pytest.raises(moe.Q36MoEError):
            call()
            raise AssertionError(f"call {i} was taken")


def test_router_calibration_step(dev):
    """The operators together, as a router and the norm in front of frozen
    quantised experts are trained on a target for the layer's output: the
    routing weights' gradient is taken from the weighted expert rows that the
    layer keeps.  Router, norm and input gradients against differentiation in
    64 bits of the same step with the same picks and expert rows."""
    T, E, k, coef, eps = 130, 32, 8, 0.02, 1e-6
    g = _g(77)
    we = synth.expert_weights(5, n_expert=E)
    experts = moe.MoEWeights.upload(we["gate"], we["up"], we["down"])
    x, a = _randn(g, T, 2048).to(dev), 0.5 * _randn(g, T, 2048).to(dev)
    nw, rw = (1 + 0.1 * _randn(g, 2048)).to(dev), (_randn(g, E, 2048) / 2048 ** 0.5).to(dev)
    mask = (torch.arange(T) < 117).to(dev)
    y, h = moe.layernorm(x, nw, a=a, eps=eps, rms=True)
    logits, _ = moe.router_logits(rw, y, E, moe.ROUTER_F32)
    idx, wt = moe.router_topk(logits, k)
    layer = moe.MoELayer(T, n_expert=E)
    layer.set_path(layer.PATH_SORTED)
    out = layer.forward(experts, y, logits, out_dtype=F32)
    target = out + _randn(g, T, 2048).to(dev) * out.std()
    dout = (out - target) * mask[:, None]
    loss, counts, psum = moe.balance_loss(logits, idx, coef=coef, mask=mask)
    rows = layer.tap(moe.TAP_DNW)[layer.tap(moe.TAP_POS).long()].view(T, k, 2048)
    dwt = (rows * dout[:, None]).sum(2) / wt
    dlogits = moe.router_topk_backward(logits, idx, dwt, counts=counts, coef=coef, mask=mask)
    drw, dy = moe.router_logits_backward(rw, y, E, dlogits)
    dres = _randn(g, T, 2048).to(dev)
    dh, dnw, _ = moe.layernorm_backward(dy, h, nw, dres=dres, eps=eps, rms=True)
    torch.cuda.synchronize()

    h64, nw64, rw64 = (t.double().cpu().requires_grad_() for t in (h, nw, rw))
    l64 = (h64 * (h64.square().mean(1, keepdim=True) + eps).rsqrt() * nw64) @ rw64.T
    q = torch.softmax(l64.gather(1, idx.long().cpu()), 1)
    live = mask.cpu()
    n = int(live.sum())
    f = counts[:E].double().cpu() / (n * k)
    aux = coef * E / n * (f * (torch.softmax(l64, 1) * live[:, None]).sum(0)).sum()
    total = (q * dwt.double().cpu() * live[:, None]).sum() + aux
    gh, gnw, grw = torch.autograd.grad(total, [h64, nw64, rw64])
    assert abs(float(loss) - float(aux.detach())) <= 1e-5 * float(aux.detach())

    def rel(got, ref):
        return float((got.double().cpu() - ref).norm() / ref.norm())

    # the logits carry 2048 fp32 roundings of values near 1 (about 1e-6), which
    # moves each probability by that much of itself; the rest is smaller
    assert rel(drw, grw) <= 2e-5 and rel(dnw, gnw) <= 2e-5
    assert rel(dh - dres, gh) <= 1e-4       # dres is 10 to 100 times larger: its rounding is in the difference
    assert not bool(dh[117:].ne(dres[117:]).any())
