"""What the sequence operators refuse: bad shapes, strides, sizes and buffers at the C ABI (checked before anything touches a
GPU) and bad tensors in Python."""
import ctypes

import pytest
import torch

from umetrack_amd import _native as nat
from umetrack_amd.lib.common import gated_filter as gf
from umetrack_amd.lib.common import row_cache as rc

P = 4096          # an address that is never dereferenced: every call below returns before a launch


def shape(**kw):
    s = nat.GatedShape(0, 4, 2, 3, 2, 12, 6, 6, 3, 12, 6, 2, 1, 2, 1, 12, 6, 6, 3)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(t=-1), dict(rows=-1), dict(groups=0), dict(share=0), dict(share=-3), dict(x_t=-1),
                                 dict(gate_row=-1), dict(valid_row=-2), dict(out_t=5), dict(out_row=5), dict(out_t=0), dict(out_row=0),
                                 dict(groups=1 << 20, share=1 << 10), dict(t=(1 << 30) + 1), dict(t=1 << 30, rows=1 << 20),
                                 dict(rows=(1 << 31) - 1, groups=1 << 10)], ids=str)
def test_scan_shapes(bad):
    L = nat.lib()
    s = shape(**bad)
    assert L.umt_gated_scan(s, P, P, None, None, None, P, None, None, None, 0, None) == 1
    assert L.umt_gated_scan_backward(s, P, P, None, None, P, P, None, P, P, None, P, 1 << 50, None) == 1
    assert L.umt_last_error()


def test_scan_pointers_and_workspaces():
    L = nat.lib()
    assert L.umt_gated_scan(None, P, P, None, None, None, P, None, None, None, 0, None) == 1
    assert L.umt_gated_scan_workspace_bytes(None) == -1 and L.umt_gated_scan_backward_workspace_bytes(None) == -1
    for k in range(3):
        a = [P, P, P]
        a[k] = None
        assert L.umt_gated_scan(shape(), a[0], a[1], None, None, None, a[2], None, None, None, 0, None) == 1
    for k in range(4):
        a = [P] * 4
        a[k] = None
        assert L.umt_gated_scan_backward(shape(), a[0], a[1], None, None, a[2], a[3], None, P, P, None, P, 1 << 40, None) == 1
    assert L.umt_gated_scan_backward(shape(dgate_t=2), P, P, None, None, P, P, None, P, P, None, P, 1 << 40, None) == 1
    wide = shape(groups=1, share=200, x_t=400, x_row=200, out_t=400, out_row=200)
    need = L.umt_gated_scan_backward_workspace_bytes(wide)
    assert need > 0
    assert L.umt_gated_scan_backward(wide, P, P, None, None, P, P, None, P, P, None, P, need - 1, None) == 5
    assert L.umt_gated_scan_backward(wide, P, P, None, None, P, P, None, P, P, None, None, need, None) == 5
    for empty in (dict(t=0), dict(rows=0), dict(t=0, rows=0)):
        assert L.umt_gated_scan_workspace_bytes(shape(**empty)) == 0 and L.umt_gated_scan_backward_workspace_bytes(shape(**empty)) == 0
    assert L.umt_gated_scan(shape(rows=0), None, None, None, None, None, None, None, None, None, 0, None) == 0


def test_step_arguments():
    L = nat.lib()

    def step(dtype=0, x=P, gate=P, idx=P, batch=3, groups=2, share=2, state=P, rows=4, out=P, ws=P, size=1 << 20):
        return L.umt_gated_step(dtype, x, gate, idx, None, None, batch, groups, share, state, rows, out, None, ws, size, None)
    for kw in (dict(dtype=5), dict(x=None), dict(gate=None), dict(out=None), dict(state=None), dict(batch=-1), dict(groups=0), dict(share=0),
               dict(rows=-1), dict(idx=None, batch=5), dict(groups=1 << 20, share=1 << 10)):
        assert step(**kw) == 1, kw
    assert step(batch=3000, rows=5000, size=8) == 5 and step(batch=3000, rows=5000, ws=None) == 5
    assert step(batch=0, x=None, gate=None, out=None) == 0


def test_strides_that_lead_out_of_memory():
    L = nat.lib()
    for bad in (dict(x_t=1 << 60), dict(gate_row=1 << 60), dict(out_t=1 << 50), dict(dh_t=(1 << 47) + 1), dict(rows=1 << 30, groups=1, share=3)):
        s = shape(**{**dict(t=4), **bad})
        assert L.umt_gated_scan_backward(s, P, P, None, None, P, P, None, P, P, None, P, 1 << 62, None) == 1, bad
    # an axis of one step or row has no stride
    assert L.umt_gated_scan(shape(t=1, x_t=1 << 60, gate_t=1 << 60, out_t=1 << 60), P, P, None, None, None, None, None, None, None, 0, None) == 1
    assert b"null pointer" in L.umt_last_error()


def test_step_places_and_sizes():
    L = nat.lib()
    x, gate, state, out = 1 << 20, 2 << 20, 3 << 20, 4 << 20          # 4 samples of 2 x 3 features, 5 rows

    def step(x=x, gate=gate, state=state, out=out, batch=4, rows=5, share=3, dtype=0, ws=P, size=1 << 40):
        return L.umt_gated_step(dtype, x, gate, P, None, None, batch, 2, share, state, rows, out, None, ws, size, None)
    for kw in (dict(out=x + 4), dict(out=x + 4 * 24 - 4), dict(out=x - 4 * 24 + 4), dict(out=gate), dict(out=gate + 4 * 8 - 4), dict(state=x),
               dict(state=x - 4 * 30 + 4), dict(state=out + 4 * 24 - 4), dict(state=gate), dict(out=gate + 4, share=1), dict(out=state + 4 * 29)):
        assert step(**kw) == 1 and b"overlap" in L.umt_last_error(), kw
    for batch, share in (((1 << 26), 1), ((1 << 31) - 1, 1), (1 << 20, 1 << 13)):
        assert step(batch=batch, share=share) == 1 and b"samples of" in L.umt_last_error()


def test_row_calls_too_large():
    L = nat.lib()
    thin, n = rows_buf((1 << 40, 4))
    big = (1 << 31) - 1
    assert L.umt_rows_copy(thin, n, 8, P, P, big, None, P, 1 << 60, None) == 1 and L.umt_rows_fork(thin, n, 8, P, P, big, P, None, P, 1 << 60, None) == 1
    long, n = rows_buf((1 << 40, 1 << 30))
    assert L.umt_rows_copy(long, n, 8, P, P, 1 << 9, None, P, 1 << 60, None) == 1 and b"pieces" in L.umt_last_error()
    assert L.umt_rows_copy_workspace_bytes(long, n, big, 1) == -1                     # more than any memory holds


def rows_buf(*entries):
    return (nat.RowBuffer * max(1, len(entries)))(*[nat.RowBuffer(p, n) for p, n in entries]), len(entries)


def test_row_arguments():
    L = nat.lib()
    good, n = rows_buf((P, 64), (P + 64 * 8, 16))
    big = 1 << 40
    for arr, k in (rows_buf(), rows_buf((None, 64)), rows_buf((P, 0)), rows_buf((P, -4)), rows_buf((P, 64), (P + 100, 16)),
                   rows_buf((P + 100, 16), (P, 64)), rows_buf(*[(P + 4096 * i, 4) for i in range(9)])):
        assert L.umt_rows_copy(arr, k, 8, P, P, 1, None, P, big, None) == 1
        assert L.umt_rows_fork(arr, k, 8, P, P, 1, P, None, P, big, None) == 1
        assert L.umt_rows_compact(arr, k, 8, P, P, P, P, big, None) == 1
        assert L.umt_rows_copy_workspace_bytes(arr, k, 8, 1) == -1
    assert L.umt_rows_copy(None, 1, 8, P, P, 1, None, P, big, None) == 1
    assert L.umt_rows_copy(good, n, 8, P, P, -1, None, P, big, None) == 1 and L.umt_rows_copy(good, n, 8, None, P, 1, None, P, big, None) == 1
    assert L.umt_rows_copy(good, n, 8, P, P, 5000, None, P, L.umt_rows_copy_workspace_bytes(good, n, 8, 5000) - 1, None) == 5
    assert L.umt_rows_copy_workspace_bytes(good, n, 8, 5000) >= 5000 * 80
    assert L.umt_rows_fork(good, n, 8, None, P, 1, P, None, P, big, None) == 1 and L.umt_rows_fork(good, n, 8, P, P, 1, None, None, P, big, None) == 1
    assert L.umt_rows_fork(good, n, 8, P, P, 9, P, None, P, 4, None) == 5
    assert L.umt_rows_compact(good, n, 8, None, P, P, P, big, None) == 1 and L.umt_rows_compact(good, n, 8, P, P, P, P, 20, None) == 5
    assert L.umt_rows_free(P, 8, None, 1, None, None) == 1 and L.umt_rows_free(None, 8, P, 1, None, None) == 1
    assert L.umt_rows_free(P, 8, P, -1, None, None) == 1 and L.umt_rows_free(P, 8, P, 0, None, None) == 0
    assert L.umt_rows_copy(good, n, 8, P, P, 0, None, None, 0, None) == 0 and L.umt_rows_fork(good, n, 8, P, P, 0, P, None, None, 0, None) == 0


@pytest.mark.parametrize("row_bytes", [1, 252, 2656])
def test_copies_into_an_empty_cache_have_their_workspace(row_bytes):
    """What the launches write whatever the row numbers are: a byte a copy where the copies are planned in LDS, a count
    and a word a copy where they are not."""
    L = nat.lib()
    for n, index in ((257, 257), (1 << 14, 1 << 14), ((1 << 14) + 1, 16 + 4 * ((1 << 14) + 1))):
        for data in (None, P):
            arr, k = rows_buf((data, row_bytes))
            need = L.umt_rows_copy_workspace_bytes(arr, k, 0, n)
            assert need >= index, (n, need)
            assert L.umt_rows_copy(arr, k, 0, P, P, n, None, P, need - 1, None) == 5
            assert L.umt_rows_copy(arr, k, 0, P, P, n, None, None, need, None) == 5


def test_model_without_rows_and_null_handles():
    L = nat.lib()
    arr, rows = (nat.RowBuffer * 2)(), ctypes.c_int(7)
    assert L.umt_model_memory_buffers(None, arr, ctypes.byref(rows)) == 1
    h = ctypes.c_void_p()
    nat.check(L.umt_model_create(ctypes.byref(h)))
    assert L.umt_model_memory_buffers(h, None, ctypes.byref(rows)) == 1 and L.umt_model_memory_buffers(h, arr, None) == 1
    assert L.umt_model_memory_buffers(h, arr, ctypes.byref(rows)) == 0 and rows.value == 0
    assert (arr[0].row_bytes, arr[1].row_bytes) == (18 * 36 * 4, 64)
    L.umt_model_destroy(h)


def test_groups_of_gates():
    def split(feat, gate):
        return gf._split("t", torch.empty((2, 3) + feat), torch.empty((2, 3) + gate), 2)
    assert split((21, 3), (21,)) == (21, 3) and split((21, 3), ()) == (1, 63) and split((21, 3), (21, 3)) == (63, 1)
    assert split((21, 3), (21, 1)) == (21, 3) and split((21, 3), (1, 1)) == (1, 63) and split((21, 3), (1,)) == (1, 63)
    assert split((18, 6, 6), (18,)) == (18, 36) and split((), ()) == (1, 1) and split((1, 3), (1,)) == (1, 3) and split((5,), (5, 1)) == (5, 1)
    for feat, gate in (((21, 3), (3,)), ((21, 3), (1, 3)), ((4,), (5,)), ((4,), (4, 2)), ((2, 3), (2, 3, 4))):
        with pytest.raises(ValueError, match="no leading dimensions"):
            split(feat, gate)
    with pytest.raises(ValueError, match="differ"):
        gf._split("t", torch.empty(2, 3, 4), torch.empty(2, 4), 2)


def test_sizes_past_31_bits():
    one = torch.empty(1, 1, 1)
    for x, gate in ((one.expand(1 << 31, 1, 1), one.expand(1 << 31, 1, 1)), (one.expand(1, 1 << 32, 1), one[:, :, 0].expand(1, 1 << 32)),
                    (one.expand(1, 1, 1 << 31), one[:, :, 0]), (one.expand(1, 1, 1 << 33), one.expand(1, 1, 1 << 33))):
        with pytest.raises(ValueError):
            gf._split("t", x, gate, 2)
    with pytest.raises(ValueError):
        rc._ids("t", torch.zeros(1, dtype=torch.int64).expand(1 << 31), torch.device("cpu"))


def test_types_and_devices():
    x, g = torch.zeros(4, 2, 3), torch.zeros(4, 2)
    for bad in ((x.half(), g.half()), (x, g.bfloat16()), (x.double(), g.double())):
        with pytest.raises(TypeError):
            gf.gated_scan(*bad)
    with pytest.raises(TypeError):
        gf.gated_scan(x.numpy(), g)
    if not torch.cuda.is_available():
        with pytest.raises(nat.UmtError, match="no MI355X"):
            gf.gated_scan(x, g)
        with pytest.raises(nat.UmtError, match="no MI355X"):
            gf.gated_step(x[0], g[0], torch.zeros(2, 3))
    with pytest.raises(ValueError):
        rc.copy_rows([torch.zeros(4, 3)], torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(TypeError):
        rc.copy_rows(["x"], torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError):
        rc.fork_rows([torch.zeros(4, 3)], torch.ones(4), torch.zeros(1, dtype=torch.int64))
    with pytest.raises(ValueError):
        rc.free_rows(torch.ones(4, dtype=torch.bool), torch.zeros(1, dtype=torch.int64))


def test_forward_mode_tangents():
    """The kernels read values alone: a dual tensor's tangent would be lost without a word."""
    from torch.autograd import forward_ad
    x, g, h0, one = torch.zeros(4, 2, 3), torch.zeros(4, 2), torch.zeros(2, 3), torch.zeros(1, dtype=torch.int64)
    kept, dh = torch.zeros(1, 6), torch.zeros(4, 2, 3)
    calls = ((lambda d: gf.gated_scan(d, g), x), (lambda d: gf.gated_scan(x, d), g), (lambda d: gf.gated_scan(x, g, h0=d), h0),
             (lambda d: gf.gated_scan(d, g, keep=True), x), (lambda d: gf.gated_step(d, g[0], h0), x[0]), (lambda d: gf.gated_step(x[0], d, h0), g[0]),
             (lambda d: gf.gated_step(x[0], g[0], d), h0), (lambda d: gf.gated_scan_backward(d, g, kept, dh), x),
             (lambda d: gf.gated_scan_backward(x, g, kept, d), dh), (lambda d: gf.gated_scan_backward(x, g, kept, dh, d), h0))
    with forward_ad.dual_level():
        for call, t in calls:
            for grad in (torch.enable_grad(), torch.no_grad()):
                with grad, pytest.raises(nat.UmtError, match="forward-mode"):
                    call(forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(Exception) as plain:            # a tensor without a tangent gets as far as it does outside
            gf.gated_scan(x, g)
        assert "forward-mode" not in str(plain.value)


def test_a_tracker_leaves_the_callers_filter_where_it_is():
    from umetrack_amd.lib.common.landmark_filter import LandmarkFilter
    from umetrack_amd.lib.tracker import tracker
    filt, other = LandmarkFilter(0.3), torch.device("meta")
    kept = list(filt.parameters())
    moved = tracker._filter_on(filt, other)
    assert moved is not filt and all(p.device == other for p in moved.parameters())
    assert all(p is q and p.device.type == "cpu" for p, q in zip(filt.parameters(), kept))
    assert tracker._filter_on(filt, torch.device("cpu")) is filt and tracker._filter_on(None, other) is None


@pytest.mark.gpu
def test_forward_mode_tangents_on_the_gpu():
    from torch.autograd import forward_ad
    d = "cuda"
    x, g, st, one = torch.rand(4, 2, 3, device=d), torch.zeros(4, 2, device=d), torch.zeros(2, 3, device=d), torch.zeros(1, dtype=torch.int64, device=d)
    want = gf.gated_scan(x, g)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: gf.gated_scan(dual, g), lambda: gf.gated_step(dual[0], g[0], st),
                     lambda: rc.copy_rows([forward_ad.make_dual(st, torch.ones_like(st))], one, one)):
            with pytest.raises(nat.UmtError, match="forward-mode"):
                call()
        assert all(torch.equal(a, b) for a, b in zip(gf.gated_scan(x, g), want))
        xr = x.clone().requires_grad_(True)
        h, _ = gf.gated_scan(xr, g)
        with pytest.raises(nat.UmtError, match="forward-mode"):
            torch.autograd.grad(h, xr, forward_ad.make_dual(torch.ones_like(h), torch.ones_like(h)))


@pytest.mark.gpu
def test_tensors_that_do_not_fit():
    d = "cuda"
    x, g = torch.zeros(4, 2, 3, device=d), torch.zeros(4, 2, device=d)
    for kw in (dict(h0=torch.zeros(2, 4, device=d)), dict(h0=torch.zeros(2, 3)), dict(h0=torch.zeros(2, 3, device=d).double()),
               dict(use_memory=torch.ones(2, 4, dtype=torch.bool, device=d)), dict(valid=torch.ones(4, 2, device=d)),
               dict(valid=torch.ones(4, 2, dtype=torch.bool))):
        with pytest.raises(ValueError):
            gf.gated_scan(x, g, **kw)
    with pytest.raises(ValueError):
        gf.gated_scan(x, g.cpu())
    with pytest.raises(ValueError):
        gf.gated_scan(x[0, 0], g[0, 0])
    st = torch.zeros(5, 3, device=d)
    for kw in (dict(state=st.double()), dict(state=st[:, :2]), dict(state=torch.zeros(5, 6, device=d)[:, ::2]), dict(state=st[:1]),
               dict(state=st, memory_idx=torch.zeros(3, dtype=torch.int64, device=d)), dict(state=st, memory_idx=torch.zeros(2, dtype=torch.int32, device=d)),
               dict(state=st, out=torch.zeros(2, 4, device=d)), dict(state=st, status=torch.zeros(2, dtype=torch.int32, device=d)),
               dict(state=st, valid=torch.ones(3, dtype=torch.bool, device=d))):
        with pytest.raises(ValueError):
            gf.gated_step(x[0], g[0], **kw)
    with pytest.raises(nat.UmtError, match="not differentiable"):
        gf.gated_step(x[0].clone().requires_grad_(True), g[0], st)
    h, last, kept = gf.gated_scan(x, g, keep=True)
    for kw in (dict(kept=kept[:0]), dict(kept=None), dict(dh=h[:2]), dict(dh=h.bfloat16()), dict(dh_last=last[:1])):
        with pytest.raises(ValueError):
            gf.gated_scan_backward(**{**dict(x=x, gate=g, kept=kept, dh=h), **kw})
    live, one = torch.ones(5, dtype=torch.bool, device=d), torch.zeros(1, dtype=torch.int64, device=d)
    for call in (lambda: rc.copy_rows([st, st[:4]], one, one), lambda: rc.copy_rows([st], one, one.int()), lambda: rc.copy_rows([st], one, one[:0]),
                 lambda: rc.copy_rows([torch.zeros(5, 6, device=d)[:, ::2]], one, one), lambda: rc.copy_rows([st], one.cpu(), one),
                 lambda: rc.copy_rows([], one, one), lambda: rc.copy_rows([st.clone() for _ in range(9)], one, one),
                 lambda: rc.fork_rows([st], live[:4], one), lambda: rc.fork_rows([st], live.int(), one), lambda: rc.compact_rows([st], live[:4]),
                 lambda: rc.free_rows(live, one.int()), lambda: rc.copy_rows([st], one, one, torch.zeros(1, device=d))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(nat.UmtError, match="overlap"):
        rc.copy_rows([st, st], one, one)
    with pytest.raises(nat.UmtError, match="gradients"):
        rc.copy_rows([st.clone().requires_grad_(True)], one, one)
    from umetrack_amd import arch
    from umetrack_amd.lib.models.model_loader import model_from_state_dict
    m = model_from_state_dict(arch.make_synthetic_state(1)).to(d)
    m.reserve_memory(3)
    with pytest.raises(ValueError, match="memory rows reserved"):
        rc.copy_rows([st, m], one, one)
