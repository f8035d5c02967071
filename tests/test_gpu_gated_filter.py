"""Gated linear recurrence (umt_gated_scan, its gradients, umt_gated_step) against its definition in 64 bits.

Tolerances.  u = 2^-24 is half a step of float32.  A step base + m (other - base) rounds three times (the difference, the
fma, m itself to about 4 u), each at most u times the largest magnitude M that the row has seen, so a step adds at most
6 u M; a later step shrinks what an earlier one left by a <= 1 - c, so the errors of all steps sum to 6 u M K with
K = min(T, 1 / min c).  Backward values obey the same recurrence with S = max |s| in M's place.  A gate's slope is the sum
over its features of c a s (h' - x), c a <= 1/4, whose factors carry those errors and a few roundings of their own.  A
bfloat16 result is rounded once more: 2^-8 of its value.
"""
import numpy as np
import pytest
import torch

from umetrack_amd import _native as nat

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _gf():
    from umetrack_amd.lib.common import gated_filter
    return gated_filter


def sigmoid(v):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-v))


def oracle(x, gate, h0, use, valid, dh=None, dh_last=None):
    """Step by step in float64; x [T,R,G,K], gate [T,R,G].  Returns h, last, and with dh also dx, dgate, dh0, s."""
    T = x.shape[0]
    use = np.ones(x.shape[:2], bool) if use is None else use
    valid = np.ones(x.shape[:2], bool) if valid is None else valid
    u4, v4 = use[..., None, None], valid[..., None, None]
    with np.errstate(invalid="ignore"):
        a = np.where(u4, np.where(v4, sigmoid(gate)[..., None], 1.0), 0.0)
        c = np.where(v4, np.where(u4, sigmoid(-gate)[..., None], 1.0), 0.0)
    xs = np.where(v4, x, 0.0)
    cur = np.zeros(x.shape[1:]) if h0 is None else h0
    h, prev = np.empty(x.shape), np.empty(x.shape)
    for t in range(T):
        prev[t] = cur
        with np.errstate(invalid="ignore"):
            cur = np.where(a[t] == 0, 0, a[t] * cur) + np.where(c[t] == 0, 0, c[t] * xs[t])
        h[t] = cur
    if dh is None:
        return h, cur
    s, v = np.empty(x.shape), (np.zeros(x.shape[1:]) if dh_last is None else dh_last)
    for t in range(T - 1, -1, -1):
        s[t] = dh[t] + v
        v = a[t] * s[t]
    dg = (np.where(u4 & v4, a * c * s * (prev - xs), 0.0)).sum(-1)
    return h, cur, c * s, dg, v, s


def make(T, R, G, K, dtype, seed, masks=True, rows_first=False, spread=1.5, nan=True):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    x = (torch.randn(T, R, G, K, generator=g) * 8 + torch.rand(1, R, G, K, generator=g) * 200).to(dt)
    gate = (torch.randn(T, R, G, generator=g) * spread + 0.5).clamp(-4, 4).to(dt)
    h0 = torch.randn(R, G, K, generator=g) * 50
    use = valid = None
    if masks:
        valid = torch.rand(T, R, generator=g) > 0.2
        use = torch.rand(T, R, generator=g) > 0.15
        if nan:
            x[~valid] = float("nan")
            gate[~valid] = float("inf")
    move = (lambda t: t.transpose(0, 1).contiguous().cuda().transpose(0, 1)) if rows_first else (lambda t: t.cuda())
    return [None if t is None else (move(t) if t.dim() > 2 and t is not h0 else t.cuda()) for t in (x, gate, h0, use, valid)]


def np64(t):
    return None if t is None else (t.cpu().numpy() if t.dtype == torch.bool else t.detach().double().cpu().numpy())


def slack(x, gate, h0, valid, T):
    """6 u M K of the module's text (masked steps hold or drop exactly and add nothing)."""
    gv, xv = np64(gate), np64(x)
    ok = np.ones(xv.shape[:2], bool) if valid is None else np64(valid)
    M = max(np.abs(xv[ok]).max(initial=0.0), 0.0 if h0 is None else float(h0.detach().abs().max()), 1e-30)
    cmin = sigmoid(-gv[ok].max(initial=0.0)) if ok.any() else 1.0
    return 6 * U * M * min(T, 1 / cmin), M, min(T, 1 / cmin)


SHAPES = [(1, 1, 1, 1), (1, 3, 21, 3), (2, 2, 22, 1), (15, 2, 21, 3), (16, 1, 1, 63), (17, 5, 7, 9), (31, 2, 1, 64), (33, 3, 5, 13),
          (64, 128, 21, 3), (65, 2, 2, 65), (100, 1, 18, 36), (257, 3, 1, 130), (640, 2, 21, 3), (1500, 1, 1, 2), (1025, 2, 3, 5),
          (48, 700, 63, 2), (5000, 2, 21, 3), (33, 100, 1, 1), (2000, 40, 1, 1), (70, 90, 5, 1), (9000, 1, 1, 70), (300, 300, 21, 3),
          (40, 30, 6, 400), (700, 3, 22, 1), (90, 700, 300, 1), (4000, 2, 40, 1), (50, 64, 18, 36), (400, 100, 21, 3),
          (300, 165, 21, 3), (290, 20, 72, 5)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("masks,rows_first", [(True, False), (True, True), (False, False)])
def test_scan_and_gradients(shape, dtype, masks, rows_first):
    T, R, G, K = shape
    x, gate, h0, use, valid = make(T, R, G, K, dtype, sum(shape), masks, rows_first)
    g = torch.Generator().manual_seed(7)
    dh = torch.randn(T, R, G, K, generator=g).to(DT[dtype]).cuda()
    dl = torch.randn(R, G, K, generator=g).cuda()
    for t in (x, gate, h0):
        t.requires_grad_(True)
    h, last = _gf().gated_scan(x, gate, h0, use, valid)
    assert h.dtype == x.dtype and last.dtype == torch.float32 and h.shape == x.shape and h.stride()[:2] == x.stride()[:2] or T == 1 or R == 1
    dx, dg, d0 = torch.autograd.grad((h, last), (x, gate, h0), (dh, dl))
    want = oracle(*map(np64, (x, gate, h0, use, valid, dh, dl)))
    eh, M, kk = slack(x, gate, h0, valid, T)
    S = max(np.abs(want[5]).max(), 1e-30)
    es = 6 * U * S * kk
    rnd = 2.0 ** -8 if dtype == "bf16" else 2 * U
    slope = K * 0.25 * (S * (eh + 4 * U * M) + 2 * M * es + 12 * U * S * 2 * M)
    for name, got, ref, tol in (("h", h, want[0], eh), ("last", last, want[1], eh), ("dx", dx, want[2], es + 4 * U * S),
                                ("dgate", dg, want[3], slope), ("dh0", d0, want[4], es)):
        got = np64(got)
        assert np.isfinite(got).all(), name
        bound = tol + (rnd if name in ("h", "dx", "dgate") else 2 * U) * np.abs(ref)
        assert (np.abs(got - ref) <= bound).all(), (name, float((np.abs(got - ref) / bound).max()))
    if dtype == "fp32":
        assert torch.equal(h.detach()[-1], last.detach())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows_first", [False, True])
def test_types_shapes_and_order_of_the_outputs(dtype, rows_first):
    for T, R, G, K in SHAPES:
        if T * R * G * K > 2_000_000:
            continue
        x, gate, h0, use, valid = make(T, R, G, K, dtype, 1, True, rows_first)
        h, last, kept = _gf().gated_scan(x, gate, h0, use, valid, keep=True)
        assert h.dtype == x.dtype and h.shape == x.shape and last.dtype == torch.float32 and last.shape == h0.shape
        assert kept.dtype == torch.float32 and kept.shape == (-(-T // nat.GATED_KEEP), R * G * K)
        assert T == 1 or R == 1 or h.stride()[:2] == x.stride()[:2]
        dx, dg, d0 = _gf().gated_scan_backward(x, gate, kept, torch.ones_like(h), last, use, valid)
        assert dx.dtype == dg.dtype == x.dtype and d0.dtype == torch.float32
        assert dx.shape == x.shape and dg.shape == gate.shape and d0.shape == h0.shape


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(3000, 2, 21, 3), (300, 20, 21, 3), (300, 200, 21, 3), (40, 1100, 63, 1), (2500, 3, 1, 63)], ids=str)
def test_the_gradient_of_a_stretched_gate(shape, dtype):
    """A filter's constants stretched over frames and rows, through every way the axis is shared out: T R slopes, each off by the
    module's bound (with gates within 0.5 of 0, so K = 1 / sigmoid(-0.5) = 2.7) and rounded to the type, then summed by torch
    (a rounding of the partial sums for each level of the sum) and rounded once more."""
    T, R, G, K = shape
    g = torch.Generator().manual_seed(sum(shape))
    x, dh = (torch.randn(T, R, G, K, generator=g).to(DT[dtype]).cuda() for _ in range(2))
    valid = (torch.rand(T, R, generator=g) > 0.1).cuda()
    use = (torch.rand(T, R, generator=g) > 0.1).cuda()
    bias = (torch.rand(G, generator=g) - 0.5).to(DT[dtype]).cuda().requires_grad_(True)
    gate = bias.expand(T, R, G)
    h, _ = _gf().gated_scan(x, gate, None, use, valid)
    (got,) = torch.autograd.grad(h, bias, dh)
    *_, slopes, _, s = oracle(*map(np64, (x, gate, None, use, valid, dh)))
    eh, M, kk = slack(x, gate, None, valid, T)
    S = np.abs(s).max()
    es = 6 * U * S * kk
    each = K * 0.25 * (S * (eh + 4 * U * M) + 2 * M * es + 12 * U * S * 2 * M)
    half_step = 2.0 ** -8 if dtype == "bf16" else U
    size = np.abs(slopes).sum((0, 1))
    want = slopes.sum((0, 1))
    tol = T * R * each + (half_step + 64 * U) * size + half_step * np.abs(want)
    assert (np.abs(np64(got) - want) <= tol).all(), float((np.abs(np64(got) - want) / tol).max())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("share", [2, 4, 6, 14, 15, 16, 17, 20, 21, 22, 28, 30, 31, 32, 33, 34, 36, 42, 47, 48, 62, 63, 64, 66, 126, 127, 128, 129, 250])
def test_gate_sums_of_every_width(share, dtype):
    """Gates that begin and end anywhere among a wave's lanes, in rows of few gates and of many."""
    for shape in ((19, 5, 7, share), (16, 3, 1, share), (3, 2, 67, share)):
        test_scan_and_gradients(shape, dtype, True, False)


def test_every_mask_combination_and_what_lies_under_it():
    """Rows that are never valid, never keep memory, or neither; NaN, infinities and the type's extremes under the masks."""
    T, R = 40, 8
    x, gate, h0, _, _ = make(T, R, 3, 5, "fp32", 1, masks=False)
    use = torch.ones(T, R, dtype=torch.bool, device="cuda")
    valid = use.clone()
    valid[:, 0] = False
    use[:, 1] = False
    valid[:, 2] = use[:, 2] = False
    valid[::2, 3] = False
    use[5, 4] = False
    valid[5, 5] = use[5, 5] = False
    valid[20:, 6] = False
    big = torch.finfo(torch.float32)
    bad = [float("nan"), float("inf"), -float("inf"), big.min, big.max]
    for i, (t, r) in enumerate((~valid).nonzero().tolist()):
        x[t, r], gate[t, r] = bad[i % 5], bad[(i + 2) % 5]
    h, last = _gf().gated_scan(x, gate, h0, use, valid)
    want, _ = oracle(*map(np64, (x, gate, h0, use, valid)))
    eh, _, _ = slack(x, gate, h0, valid, T)
    got = np64(h)
    assert np.isfinite(got).all() and (np.abs(got - want) <= eh + 2 * U * np.abs(want)).all()
    assert torch.equal(h[:, 0], h0[0].expand(T, 3, 5)) and torch.equal(h[:, 1], x[:, 1])
    assert bool((h[:, 2] == 0).all()) and torch.equal(last[6], h[-1, 6])
    # A skipped frame's exact value is its predecessor's.  Two frames of different stretches reach it by different orders of the
    # same steps, each within eh of it, so they lie within 2 eh of each other; within a stretch they are the same bits.
    assert float((h[20:, 6] - h[19:20, 6]).abs().max()) <= 2 * eh and torch.equal(h[32:, 6], h[32:33, 6].expand(8, 3, 5))


def test_gates_at_their_ends_and_a_poisoned_memory():
    """gate = +-inf and the type's extremes hold or replace exactly; a memory of NaN is gone where it is dropped."""
    inf, big = float("inf"), torch.finfo(torch.float32).max
    gate = torch.tensor([inf, -inf, big, -big, 200.0, -200.0, 0.0], device="cuda")[:, None, None].expand(7, 2, 1)
    x = torch.arange(1.0, 8.0, device="cuda")[:, None, None].expand(7, 2, 3).contiguous()
    h0 = torch.full((2, 3), 100.0, device="cuda")
    h, _ = _gf().gated_scan(x, gate, h0)
    assert h[:, 0, 0].tolist() == [100.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.5]
    h0[1] = float("nan")
    use = torch.ones(7, 2, dtype=torch.bool, device="cuda")
    use[0] = False
    h, _ = _gf().gated_scan(x, torch.zeros(7, 2, device="cuda"), h0, use_memory=use)
    assert bool(torch.isfinite(h).all()) and torch.equal(h[:, 0], h[:, 1]) and h[0, 0, 0] == 1.0
    st = h0.clone()
    _gf().gated_step(x[0], torch.zeros(2, device="cuda"), st, use_memory=use[0])
    assert torch.equal(st, x[0])


RANGE_SHAPES = [(1, 2, 3, 2), (40, 3, 5, 3), (300, 20, 21, 3), (3000, 2, 7, 4), (40, 1100, 63, 1)]     # alone, tiles, runs


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", RANGE_SHAPES, ids=str)
@pytest.mark.parametrize("masks", [True, False])
def test_values_at_the_ends_of_the_range(shape, dtype, masks):
    """Inputs and states of either sign up to 3e38: their differences are beyond the largest float, the mix is not.  The
    tolerances are the module's with M = 3e38; gradients small enough that no slope (a quarter of the difference times s) leaves
    the range."""
    T, R, G, K = shape
    _, gate, _, use, valid = make(T, R, G, K, dtype, 3 * sum(shape), masks)
    g = torch.Generator().manual_seed(1)
    sign = lambda *s: torch.randint(0, 2, s, generator=g) * 2.0 - 1
    x = (sign(T, R, G, K) * (2e38 + 1e38 * torch.rand(T, R, G, K, generator=g))).to(DT[dtype]).cuda()
    h0 = (sign(R, G, K) * 3e38).cuda()
    dh = (1e-4 * torch.randn(T, R, G, K, generator=g)).to(DT[dtype]).cuda()
    dl = (1e-4 * torch.randn(R, G, K, generator=g)).cuda()
    before, gate_of = h0[:, :, :].clone(), gate.detach()
    for t in (x, gate, h0):
        t.requires_grad_(True)
    h, last = _gf().gated_scan(x, gate, h0, use, valid)
    grads = torch.autograd.grad((h, last), (x, gate, h0), (dh, dl))
    want = oracle(*map(np64, (x, gate, h0, use, valid, dh, dl)))
    eh, M, kk = slack(x, gate, h0, valid, T)
    S = np.abs(want[5]).max()
    es = 6 * U * S * kk
    rnd = 2.0 ** -8 if dtype == "bf16" else 2 * U
    slope = K * 0.25 * (S * (eh + 4 * U * M) + 2 * M * es + 12 * U * S * 2 * M)
    assert np.abs(want[3]).max() < 3e38
    for name, got, ref, tol in (("h", h, want[0], eh), ("last", last, want[1], eh), ("dx", grads[0], want[2], es + 4 * U * S),
                                ("dgate", grads[1], want[3], slope), ("dh0", grads[2], want[4], es)):
        got = np64(got)
        assert np.isfinite(got).all(), name
        assert (np.abs(got - ref) <= tol + (rnd if name in ("h", "dx", "dgate") else 2 * U) * np.abs(ref)).all(), name
    with torch.no_grad():
        one, _ = _gf().gated_scan(x[:1], gate_of[:1], before, None if use is None else use[:1], None if valid is None else valid[:1])
        out = _gf().gated_step(x[0].detach(), gate_of[0], before, use_memory=None if use is None else use[0], valid=None if valid is None else valid[0])
    assert torch.equal(out, one[0]) and bool(torch.isfinite(before).all())


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 2, 1, 2), (40, 2, 1, 2), (300, 20, 21, 3), (3000, 2, 1, 2), (40, 1100, 63, 1)], ids=str)
def test_an_infinite_state_is_kept_while_frames_are_skipped_and_mixed_as_the_formula_says(shape, dtype):
    """In the first feature: an infinite h0, all frames skipped in row 0; frames that count in row 1, where an infinity of the
    other sign then meets it (NaN) and the memory is dropped after that.  In the last one: an infinite input, whichever
    weight is the larger."""
    T, R, G, K = shape
    x, gate, h0, _, _ = make(T, R, G, K, "fp32", T, masks=False)
    use, valid = (torch.ones(T, R, dtype=torch.bool, device="cuda") for _ in range(2))
    valid[:, 0] = False
    x[:, 0], gate[:, 0] = float("nan"), float("nan")
    h0[0, 0, 0], h0[1, 0, 0] = float("inf"), -float("inf")
    if T > 20:
        x[T // 2, 1, 0, 0] = float("inf")
        use[T - T // 4, 1] = False
        x[T // 3, 1, 0, K - 1] = -float("inf") if K > 1 else x[T // 3, 1, 0, 0]
    x, gate = x.to(DT[dtype]), gate.to(DT[dtype])
    state = h0.clone()
    h, last = _gf().gated_scan(x, gate, h0, use, valid)
    want, wl = oracle(*map(np64, (x, gate, h0, use, valid)))
    assert np.isposinf(want[:, 0, 0, 0]).all() and np.isneginf(want[0, 1, 0, 0])
    kind = lambda v: np.where(np.isnan(v), 3, np.where(np.isposinf(v), 2, np.where(np.isneginf(v), 1, 0)))
    assert np.array_equal(kind(np64(h)), kind(want)) and np.array_equal(kind(np64(last)), kind(wl))
    ok = np.isfinite(want)
    h0f = torch.nan_to_num(h0, 0, 0, 0)
    xf = torch.nan_to_num(x.float(), 0, 0, 0)
    eh, _, _ = slack(xf, gate, h0f, valid, T)
    assert (np.abs(np64(h)[ok] - want[ok]) <= eh + (2.0 ** -8 if dtype == "bf16" else 2 * U) * np.abs(want[ok])).all()
    for t in range(min(T, 3)):
        out = _gf().gated_step(x[t], gate[t], state, use_memory=use[t], valid=valid[t])
        assert np.array_equal(kind(np64(out)), kind(want[t]))


def test_slow_memory_and_old_outliers_keep_their_precision():
    """c = 8e-7 over 20000 frames: the response to a constant is 1 - a^T up to the rounding of the state, T u of it (1.2e-3);
    rounding a itself would change c by up to u / c = 7 % of it.  An outlier of 1e6 ahead of values
    around 1 is forgotten to 20 u of what is left of it and of the values."""
    T = 20000
    x = torch.ones(T, 2, 3, device="cuda")
    gate = torch.full((1, 1), 14.0, device="cuda").expand(T, 2)
    h, last = _gf().gated_scan(x, gate)
    c = sigmoid(-14.0)
    want = -np.expm1(np.arange(1, T + 1) * np.log1p(-c))
    assert (np.abs(np64(h)[:, 0, 0] - want) <= (np.arange(1, T + 1) + 8) * U * want).all()
    T = 600
    x = 1 + torch.rand(T, 2, 3, device="cuda")
    h0 = torch.full((2, 3), 1e6, device="cuda")
    for g in (-2.0, 0.0, 2.0):
        gate = torch.full((T, 2), g, device="cuda")
        h, _ = _gf().gated_scan(x, gate, h0)
        a = sigmoid(g)
        left = 1e6 * a ** np.arange(1, T + 1)
        want, _ = oracle(np64(x)[:, :, None], np64(gate)[..., None], np64(h0)[:, None], None, None)
        steps = np.arange(1, T + 1)
        bound = (20 + 6 * np.minimum(steps, 1 / (1 - a))) * U * 2 + 6 * U * steps * left
        assert (np.abs(np64(h) - want[:, :, 0]).max((1, 2)) <= bound).all(), g


def test_gradient_against_differences():
    """<gradient, d> against central differences of the 64-bit definition: their own error is eps^2 |f'''| + 1e-16 |f| / eps."""
    T, R, G, K = 37, 3, 4, 3
    x, gate, h0, use, valid = make(T, R, G, K, "fp32", 3, nan=False)
    for t in (x, gate, h0):
        t.requires_grad_(True)
    g = torch.Generator().manual_seed(5)
    w, wl = torch.randn(T, R, G, K, generator=g), torch.randn(R, G, K, generator=g)
    h, last = _gf().gated_scan(x, gate, h0, use, valid)
    grads = torch.autograd.grad((h * w.cuda()).sum() + (last * wl.cuda()).sum(), (x, gate, h0))
    un, vn = np64(use), np64(valid)

    def loss(a, b, c):
        hh, ll = oracle(a, b, c, un, vn)
        return (hh * w.double().numpy()).sum() + (ll * wl.double().numpy()).sum()
    base = [np64(t) for t in (x, gate, h0)]
    rng = np.random.default_rng(0)
    for k in range(3):
        d = rng.standard_normal(base[k].shape)
        eps = 1e-5
        up, dn = list(base), list(base)
        up[k], dn[k] = base[k] + eps * d, base[k] - eps * d
        num = (loss(*up) - loss(*dn)) / (2 * eps)
        ana = float((np64(grads[k]) * d).sum())
        scale = float((np.abs(np64(grads[k])) * np.abs(d)).sum())
        assert abs(num - ana) <= 3e-6 * scale, (k, num, ana, scale)


def test_strides_offsets_and_broadcast_gates():
    """Padded rows, an odd storage offset, features that are no run of memory, an expanded gate whose gradient torch sums."""
    T, R, G, K = 50, 6, 5, 3
    x, gate, h0, use, valid = make(T, R, G, K, "fp32", 11)
    ref, rl = _gf().gated_scan(x, gate, h0, use, valid)
    wide = torch.full((T, R + 2, 40), 9.0, device="cuda")
    xv = wide.view(-1)[7:].as_strided((T, R, G, K), ((R + 2) * 40, 40, K, 1))
    xv.copy_(x)
    swapped = x.transpose(2, 3).contiguous().transpose(2, 3)
    big = torch.zeros(T, R, 2 * G, device="cuda")
    big[:, :, ::2] = gate
    mk = torch.zeros(R, T, 3, dtype=torch.bool, device="cuda")
    mk[:, :, 1] = use.t()
    for a, b, m in ((xv, gate, use), (swapped, gate, use), (x, big[:, :, ::2], use), (x, gate, mk[:, :, 1].t())):
        h, last = _gf().gated_scan(a, b, h0, m, valid)
        assert torch.equal(h, ref) and torch.equal(last, rl)
    for dt in (torch.float32, torch.bfloat16):
        one = torch.tensor([0.3], device="cuda", dtype=dt, requires_grad=True)
        y = torch.randn(T, R, G, K, device="cuda").to(dt)
        h, _ = _gf().gated_scan(y, one.expand(T, R, 1))
        dh = torch.randn(T, R, G, K, device="cuda").to(dt)
        (got,) = torch.autograd.grad(h, one, dh)
        *_, want, _, s = oracle(np64(y).reshape(T, R, 1, G * K), np.full((T, R, 1), float(one.detach())), None, None, None,
                                np64(dh).reshape(T, R, 1, G * K))
        # T R slopes rounded to the type, then summed by torch and rounded again
        tol = 2 * torch.finfo(dt).eps * np.abs(want).sum() + 40 * U * np.abs(want).sum() + 2.0 ** -16 * T * R
        assert abs(float(got) - want.sum()) <= tol


def test_only_the_gradients_that_are_asked_for():
    x, gate, h0, use, valid = make(70, 3, 2, 70, "fp32", 2)
    xg = x.clone().requires_grad_(True)
    h, last = _gf().gated_scan(xg, gate, h0, use, valid)
    (a,) = torch.autograd.grad(last.sum(), xg, retain_graph=True)
    (b,) = torch.autograd.grad(h[-1].sum(), xg)
    # the same gradient, which enters the last stretch from behind or at its last step: two orders of the same steps, each
    # within 6 u S K + 4 u S of it, and S = 1 here
    _, _, kk = slack(x, gate, h0, valid, 70)
    assert float((a - b).abs().max()) <= 2 * (6 * U * kk + 4 * U)
    h, last, kept = _gf().gated_scan(x, gate, h0, use, valid, keep=True)
    dh = torch.randn_like(h)
    full = _gf().gated_scan_backward(x, gate, kept, dh, None, use, valid)
    for i in range(3):
        part = _gf().gated_scan_backward(x, gate, kept, dh, None, use, valid, need=tuple(j == i for j in range(3)))
        assert torch.equal(part[i], full[i]) and [p is None for p in part] == [j != i for j in range(3)]
    assert bool((full[0][~valid] == 0).all()) and bool((full[1][~(valid & use)] == 0).all())


def test_empty_axes():
    gf = _gf()
    h0 = torch.randn(3, 4, device="cuda")
    h, last = gf.gated_scan(torch.empty(0, 3, 4, device="cuda"), torch.empty(0, 3, device="cuda"), h0)
    assert h.shape == (0, 3, 4) and torch.equal(last, h0)
    assert bool((gf.gated_scan(torch.empty(0, 3, 4, device="cuda"), torch.empty(0, 3, device="cuda"))[1] == 0).all())
    a, b, c = (t.requires_grad_(True) for t in (torch.empty(0, 3, 4, device="cuda"), torch.empty(0, 3, device="cuda"), h0))
    h, last = gf.gated_scan(a, b, c)
    assert torch.equal(torch.autograd.grad(last, c, h0.detach() * 2)[0], h0.detach() * 2)
    for shape in ((5, 0, 4), (5, 3, 0)):
        h, last = gf.gated_scan(torch.empty(shape, device="cuda"), torch.empty(shape[:2], device="cuda"))
        assert h.shape == shape and last.shape == shape[1:]
    st = torch.ones(4, 2, device="cuda")
    assert gf.gated_step(torch.empty(0, 2, device="cuda"), torch.empty(0, device="cuda"), st).shape == (0, 2) and bool((st == 1).all())


def test_offsets_past_32_bits():
    """Steps 2^30 + 37 elements apart: the third lies past 2^31."""
    step = (1 << 30) + 37
    big = torch.empty(2 * step + 64, dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((3, 2, 30), (step, 32, 1))
    vals = torch.randn(3, 2, 30, device="cuda").bfloat16()
    x.copy_(vals)
    gate = torch.randn(3, 2, device="cuda").bfloat16()
    h, last = _gf().gated_scan(x, gate)
    ref, rl = _gf().gated_scan(vals, gate)
    assert torch.equal(h, ref) and torch.equal(last, rl)


def test_rows_further_apart_than_32_bits():
    """Rows 2^30 + 5 elements apart, their features two wide: a wave holds values of all three rows."""
    far = (1 << 30) + 5
    big = torch.empty(2 * far + 4096, dtype=torch.float32, device="cuda")
    for T in (5, 900):
        x = big.as_strided((T, 3, 2), (2, far, 1))
        vals = torch.randn(T, 3, 2, device="cuda")
        x.copy_(vals)
        gate, valid = torch.randn(T, 3, 2, device="cuda"), torch.rand(T, 3, device="cuda") > 0.3
        h, last, kept = _gf().gated_scan(x, gate, valid=valid, keep=True)
        ref, rl, rk = _gf().gated_scan(vals, gate, valid=valid, keep=True)
        assert torch.equal(h, ref) and torch.equal(last, rl) and torch.equal(kept, rk)
        dh = torch.randn(T, 3, 2, device="cuda")
        for a, b in zip(_gf().gated_scan_backward(x, gate, kept, dh, valid=valid), _gf().gated_scan_backward(vals, gate, rk, dh, valid=valid)):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T", [700, 6000, 20011])
def test_masks_across_stretches_and_segments(T):
    """Long runs of skipped frames, a memory dropped once in a long while, NaN memory dropped late, NaN below every mask."""
    R, G, K = 4, 5, 3
    x, gate, h0, _, _ = make(T, R, G, K, "fp32", T, masks=False)
    gate += 3
    gate[:, 2] = 12.0
    use, valid = (torch.ones(T, R, dtype=torch.bool, device="cuda") for _ in range(2))
    valid[T // 7:T - 5, 0] = False
    use[[0, T // 3, T // 3 + 1, T - 1], 1] = False
    valid[::3, 2] = False
    use[T // 2, 3] = False
    valid[T // 2 + 1:, 3] = False
    use[1, 2] = False
    h0[1] = float("nan")
    h0[2] = float("inf")
    valid[0, 2], use[0, 2] = False, False
    x[~valid] = float("nan")
    gate[~valid] = float("nan")
    for t in (x, gate, h0):
        t.requires_grad_(True)
    g = torch.Generator().manual_seed(1)
    dh, dl = torch.randn(T, R, G, K, generator=g).cuda(), torch.randn(R, G, K, generator=g).cuda()
    h, last = _gf().gated_scan(x, gate, h0, use, valid)
    got = (h, last) + torch.autograd.grad((h, last), (x, gate, h0), (dh, dl))
    h0d = np.nan_to_num(np64(h0), nan=0, posinf=0)
    ref = oracle(np64(x), np64(gate), h0d, np64(use), np64(valid), np64(dh), np64(dl))
    eh, M, kk = slack(x, gate, torch.from_numpy(h0d), valid, T)
    S = np.abs(ref[5]).max()
    es = 6 * U * S * kk
    tols = (eh, eh, es + 4 * U * S, K * 0.25 * (S * (eh + 4 * U * M) + 2 * M * es + 12 * U * S * 2 * M), es)
    for name, a, b, tol in zip(("h", "last", "dx", "dgate", "dh0"), got, ref, tols):
        a = np64(a)
        assert np.isfinite(a).all() and (np.abs(a - b) <= tol + 2 * U * np.abs(b)).all(), name


@pytest.mark.parametrize("T", [40, 3000])
def test_what_is_not_finite_stays_in_its_feature_until_the_memory_is_dropped(T):
    """A NaN or infinite input, gate or state that no mask excludes: its feature is not finite from there to the drop, in
    every stretch and run on the way, and no other feature notices.  Infinite gates hold or replace."""
    R, G, K = 3, 4, 2
    x, gate, h0, _, _ = make(T, R, G, K, "fp32", T, masks=False)
    clean, _ = _gf().gated_scan(x, gate, h0)
    drop = 3 * T // 4
    use = torch.ones(T, R, dtype=torch.bool, device="cuda")
    use[drop] = False
    dropped, _ = _gf().gated_scan(x, gate, h0, use)
    x[T // 8, 0, 1, 0] = float("nan")
    x[T // 8, 0, 2, 1] = float("inf")
    gate[T // 4, 1, 3] = float("nan")
    h0[2, 0, 0] = -float("inf")
    h, last = _gf().gated_scan(x, gate, h0, use)
    bad = torch.zeros(T, R, G, K, dtype=torch.bool, device="cuda")
    bad[T // 8:drop, 0, 1, 0] = bad[T // 8:drop, 0, 2, 1] = bad[:drop, 2, 0, 0] = True
    bad[T // 4:drop, 1, 3] = True
    assert torch.equal(~torch.isfinite(h), bad) and bool(torch.isfinite(last).all())
    assert torch.equal(h[~bad], dropped[~bad]) and torch.equal(dropped[:drop], clean[:drop])
    gate = torch.full((T, R), float("inf"), device="cuda")
    gate[T // 2] = -float("inf")
    x = torch.rand(T, R, K, device="cuda")
    h, _ = _gf().gated_scan(x, gate, h0[:, 0].nan_to_num(0, 0, 0))
    assert torch.equal(h[T // 2:], x[T // 2].expand(T - T // 2, R, K))


def test_other_stream_and_graph_replays():
    """Forward and backward captured into one graph, replayed with new contents between eager work and synchronisations."""
    gf = _gf()
    shape = (130, 4, 21, 3)
    x, gate, h0, use, valid = make(*shape, "fp32", 21)
    dh = torch.randn(shape, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = gf.gated_scan(x, gate, h0, use, valid, keep=True)
        ga = gf.gated_scan_backward(x, gate, a[2], dh, None, use, valid)
    torch.cuda.current_stream().wait_stream(side)
    b = gf.gated_scan(x, gate, h0, use, valid, keep=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    state = torch.zeros(8, 21, 3, device="cuda")
    idx = torch.tensor([5, 1, 7, 5], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, last, kept = gf.gated_scan(x, gate, h0, use, valid, keep=True)
        grads = gf.gated_scan_backward(x, gate, kept, dh, None, use, valid)
        frame = gf.gated_step(x[0], gate[0], state, memory_idx=idx, use_memory=use[0], valid=valid[0])
    del ga
    for k in range(4):
        y, gg, hh, uu, vv = make(*shape, "fp32", 30 + k)
        for t, n in ((x, y), (gate, gg), (h0, hh), (use, uu), (valid, vv)):
            t.copy_(n)
        state.fill_(float(k))
        eager_state = state.clone()
        graph.replay()
        e = gf.gated_scan(x, gate, h0, use, valid, keep=True)
        eg = gf.gated_scan_backward(x, gate, e[2], dh, None, use, valid)
        ef = gf.gated_step(x[0], gate[0], eager_state, memory_idx=idx, use_memory=use[0], valid=valid[0])
        torch.cuda.synchronize()
        assert torch.equal(h, e[0]) and torch.equal(last, e[1])
        assert all(torch.equal(p, q) for p, q in zip(grads, eg))
        assert torch.equal(frame, ef) and torch.equal(state, eager_state)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,rows,G,K", [(1, 1, 21, 3), (2, 2, 21, 3), (5, 9, 1, 1), (70, 300, 7, 9), (3, 5, 648, 1), (3000, 4096, 18, 36), (260, 260, 5, 64)])
def test_step_is_one_step_of_the_scan(B, rows, G, K, dtype):
    x, gate, _, use, valid = make(1, B, G, K, dtype, B + rows)
    x, gate, use, valid = x[0], gate[0], use[0], valid[0]
    g = torch.Generator().manual_seed(1)
    state = (torch.randn(rows, G, K, generator=g) * 50).cuda()
    idx = torch.randperm(rows, generator=g)[:B].cuda()
    before = state.clone()
    out = _gf().gated_step(x, gate, state, memory_idx=idx, use_memory=use, valid=valid)
    h, last = _gf().gated_scan(x[None], gate[None], before[idx], use[None], valid[None])
    assert torch.equal(out, h[0]) and torch.equal(state[idx], last)
    rest = torch.ones(rows, dtype=torch.bool, device="cuda")
    rest[idx] = False
    assert torch.equal(state[rest], before[rest])
    again = before.clone()
    out = _gf().gated_step(x, gate, again[:B], valid=valid)
    h, last = _gf().gated_scan(x[None], gate[None], before[:B], None, valid[None])
    assert torch.equal(out, h[0]) and torch.equal(again[:B], last) and torch.equal(again[B:], before[B:])


@pytest.mark.parametrize("B,spread", [(6, 2), (1000, 3), (1000, 700), (5000, 40), (20000, 9000)])
def test_step_duplicates_and_indices_outside_the_cache(B, spread):
    rows, G, K = 10000, 3, 5
    g = torch.Generator().manual_seed(B)
    x, gate = torch.randn(B, G, K, generator=g).cuda(), torch.randn(B, G, generator=g).cuda()
    use = (torch.rand(B, generator=g) > 0.2).cuda()
    idx = torch.randint(0, spread, (B,), generator=g)
    idx[::17] = rows
    idx[::19] = -1
    idx[::23] = -(1 << 40)
    idx = idx.cuda()
    state = torch.randn(rows, G, K, generator=g).cuda()
    before, status = state.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
    out = _gf().gated_step(x, gate, state, memory_idx=idx, use_memory=use, status=status)
    ok = (idx >= 0) & (idx < rows)
    h, last = _gf().gated_scan(x[None], gate[None], before[idx.clamp(0, rows - 1)], (use & ok)[None])
    assert torch.equal(out, h[0]) and int(status) == nat.STATUS_BAD_MEMORY_IDX
    want = before.clone()
    hi = {}
    for b, r in enumerate(idx.tolist()):
        if 0 <= r < rows:
            hi[r] = b
    want[torch.tensor(list(hi), device="cuda")] = last[torch.tensor(list(hi.values()), device="cuda")]
    assert torch.equal(state, want)


def test_steps_follow_the_scan():
    """A recording stepped frame by frame, as the tracker does, against the scan of it: both hold the 64-bit tolerance."""
    T, R, G, K = 90, 4, 21, 3
    x, gate, h0, use, valid = make(T, R, G, K, "fp32", 8)
    state = h0.clone()
    outs = torch.stack([_gf().gated_step(x[t], gate[t], state, use_memory=use[t], valid=valid[t]) for t in range(T)])
    h, last = _gf().gated_scan(x, gate, h0, use, valid)
    eh, _, _ = slack(x, gate, h0, valid, T)
    assert float((outs - h).abs().max()) <= 2 * eh and float((state - last).abs().max()) <= 2 * eh


def test_gates_of_no_features_have_no_gradient():
    x, g = torch.zeros(3, 2, 21, 0, device="cuda", requires_grad=True), torch.randn(3, 2, 21, device="cuda", requires_grad=True)
    torch.full((3, 2, 21), float("nan"), device="cuda")          # what the allocator hands out next
    h, last = _gf().gated_scan(x, g)
    (h.sum() + last.sum()).backward()
    assert h.shape == x.shape and x.grad.shape == x.shape and torch.equal(g.grad, torch.zeros_like(g))


@pytest.mark.parametrize("share", [1, 3])
def test_a_step_in_place(share):
    gen = torch.Generator().manual_seed(5)
    x, gate, state = torch.randn(40, 7 * share, generator=gen), torch.randn(40, 7, generator=gen), torch.randn(30, 7 * share, generator=gen)
    idx = torch.randint(-2, 30, (40,), generator=gen)
    x = x.view(40, 7, share).to("cuda")
    a, b = state.view(30, 7, share).to("cuda"), state.view(30, 7, share).to("cuda").clone()
    want = _gf().gated_step(x, gate.to("cuda"), a, memory_idx=idx.to("cuda"))
    y = x.clone()
    assert _gf().gated_step(y, gate.to("cuda"), b, memory_idx=idx.to("cuda"), out=y) is y
    assert torch.equal(y, want) and torch.equal(a, b)
    few = dict(gate=gate[:10].to("cuda"), memory_idx=idx[:10].to("cuda"))
    for kw in (dict(x=x[:10], out=b[5:15]), dict(x=b[5:15], out=torch.empty_like(b[5:15])), dict(x=y[:10], out=y[1:11])):
        with pytest.raises(nat.UmtError, match="overlap"):
            _gf().gated_step(state=b, **few, **kw)
