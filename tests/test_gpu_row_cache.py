"""Rows of state caches (umt_rows_copy / fork / free / compact) against the same operations on host lists: values are moved,
so everything is compared exactly."""
import numpy as np
import pytest
import torch

from umetrack_amd import _native as nat

pytestmark = pytest.mark.gpu

# row shapes and types: the model's and the filter's rows, odd byte counts, an int64, a long row
KINDS = {"tracker": [((18, 6, 6), torch.float32), ((4, 4), torch.float32), ((21, 3), torch.float32)],
         "odd": [((3,), torch.uint8), ((5,), torch.bfloat16), ((), torch.int64), ((7, 3), torch.float32)],
         "long": [((9001,), torch.float32), ((13000,), torch.uint8)]}


def _rc():
    from umetrack_amd.lib.common import row_cache
    return row_cache


def buffers(kind, rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for shape, dt in KINDS[kind]:
        t = torch.randint(0, 120, (rows,) + shape, generator=g).to(dt)
        out.append(t.cuda())
    return out


def host(bufs):
    return [b.cpu().clone() for b in bufs]


def same(bufs, want):
    return all(torch.equal(b.cpu(), w) for b, w in zip(bufs, want))


def status():
    return torch.zeros(1, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("kind,rows,n", [("tracker", 2, 2), ("tracker", 64, 13), ("odd", 33, 33), ("odd", 1, 1), ("long", 9, 7),
                                         ("tracker", 3000, 2500), ("odd", 20000, 19999), ("tracker", 40, 200),
                                         ("odd", 200000, 3000), ("odd", 300000, 900), ("long", 60, 50)])
@pytest.mark.parametrize("how", ["any", "permutation", "apart"])
def test_copy_reads_before_it_writes(kind, rows, n, how):
    bufs = buffers(kind, rows)
    want = host(bufs)
    g = torch.Generator().manual_seed(n)
    if how == "any":
        src, dst = torch.randint(0, rows, (n,), generator=g), torch.randint(0, rows, (n,), generator=g)
    elif how == "permutation":
        n = min(n, rows)
        dst = torch.randperm(rows, generator=g)[:n]
        src = dst[torch.randperm(n, generator=g)]
    else:
        n = min(n, rows // 2)
        p = torch.randperm(rows, generator=g)
        src, dst = p[:n], p[rows - n:]
    old = [w.clone() for w in want]
    for s, d in zip(src.tolist(), dst.tolist()):
        for w, o in zip(want, old):
            w[d] = o[s]
    st = status()
    _rc().copy_rows(bufs, src.cuda(), dst.cuda(), st)
    assert same(bufs, want) and int(st) == 0


def test_copy_skips_rows_outside_the_cache():
    bufs = buffers("tracker", 10)
    want = host(bufs)
    src, dst = [0, 10, 3, -1, 4, 1 << 40, 5], [1, 2, 11, 4, -7, 6, 5]
    old = want[0][0].clone(), want[1][0].clone(), want[2][0].clone()
    for w, o in zip(want, old):
        w[1] = o
    st = status()
    _rc().copy_rows(bufs, torch.tensor(src).cuda(), torch.tensor(dst).cuda(), st)
    assert same(bufs, want) and int(st) == nat.STATUS_BAD_ROW


@pytest.mark.parametrize("kind,rows,n", [("tracker", 10, 20), ("tracker", 900, 3000), ("odd", 200000, 3000), ("odd", 5000, (1 << 14) + 5),
                                         ("odd", (1 << 18) + 9, 3000)])
def test_every_form_of_the_copy_skips_rows_outside_the_cache(kind, rows, n):
    """A few rows, copies planned in LDS, a table of the cache.  A third of the pairs has a bad source or target; targets are
    named twice, and of some the highest copy is a bad one, which then does not count."""
    bufs = buffers(kind, rows)
    want = host(bufs)
    old = [w.clone() for w in want]
    g = torch.Generator().manual_seed(rows + n)
    src, dst = torch.randint(0, rows, (n,), generator=g), torch.randint(0, min(rows, n // 3 + 1), (n,), generator=g)
    bad = torch.tensor([-1, rows, rows + 7, 1 << 40, -(1 << 40)])
    for t in (src, dst):
        at = torch.rand(n, generator=g) < 0.18
        t[at] = bad[torch.randint(0, 5, (int(at.sum()),), generator=g)]
    half = torch.arange(n // 2, n)[:max(1, n // 20)]
    dst[half + (n - n // 2) // 2] = dst[half]              # the second of these is the higher one, and its source is bad
    src[half + (n - n // 2) // 2] = rows
    for s, d in zip(src.tolist(), dst.tolist()):
        if 0 <= s < rows and 0 <= d < rows:
            for w, o in zip(want, old):
                w[d] = o[s]
    st = status()
    _rc().copy_rows(bufs, src.cuda(), dst.cuda(), st)
    assert same(bufs, want) and int(st) == nat.STATUS_BAD_ROW
    bufs = buffers(kind, rows)
    _rc().copy_rows(bufs, src.cuda(), dst.cuda())                            # without a status word
    assert same(bufs, want)


@pytest.mark.parametrize("kind,rows,n,dead", [("tracker", 4, 2, 2), ("tracker", 64, 5, 9), ("odd", 1000, 300, 300), ("odd", 1025, 100, 40),
                                              ("tracker", 5000, 1500, 2000), ("long", 9, 3, 4), ("odd", 70000, 30000, 33000), ("odd", 5, 3, 0)])
def test_free_and_fork(kind, rows, n, dead):
    bufs = buffers(kind, rows)
    want = host(bufs)
    g = torch.Generator().manual_seed(rows)
    live = torch.ones(rows, dtype=torch.bool, device="cuda")
    drop = torch.randperm(rows, generator=g)[:dead]
    st = status()
    _rc().free_rows(live, drop.cuda(), st)
    _rc().free_rows(live, torch.cat([drop, drop]).cuda(), st)                # twice is as once
    mirror = torch.ones(rows, dtype=torch.bool)
    mirror[drop] = False
    assert torch.equal(live.cpu(), mirror) and int(st) == 0
    src = torch.randint(0, rows, (n,), generator=g)                          # some of them free, some twice
    want_ids, bad = [], 0
    free_rows = [r for r in range(rows) if not mirror[r]]
    was = mirror.clone()
    short = 0
    for s in src.tolist():
        if not was[s]:
            want_ids.append(-1)
            bad = nat.STATUS_BAD_ROW
        elif free_rows:
            r = free_rows.pop(0)
            want_ids.append(r)
            mirror[r] = True
            for w in want:
                w[r] = w[s]
        else:
            want_ids.append(-1)
            short = nat.STATUS_NO_FREE_ROW
    ids = _rc().fork_rows(bufs, live, src.cuda(), st)
    assert ids.tolist() == want_ids and torch.equal(live.cpu(), mirror) and same(bufs, want)
    assert int(st) == bad | short


def test_rows_outside_the_cache_are_neither_freed_nor_forked():
    bufs = buffers("tracker", 6)
    want = host(bufs)
    live = torch.tensor([1, 1, 0, 1, 1, 0], dtype=torch.bool, device="cuda")
    st = status()
    _rc().free_rows(live, torch.tensor([-1, 6, 1 << 40], device="cuda"), st)
    assert live.tolist() == [True, True, False, True, True, False] and int(st) == nat.STATUS_BAD_ROW
    st.zero_()
    ids = _rc().fork_rows(bufs, live, torch.tensor([-3, 0, 6, 4, 2, 3], device="cuda"), st)
    assert ids.tolist() == [-1, 2, -1, 5, -1, -1] and bool(live.all())
    for w in want:
        w[2], w[5] = w[0], w[4]
    assert same(bufs, want) and int(st) == nat.STATUS_BAD_ROW | nat.STATUS_NO_FREE_ROW


@pytest.mark.parametrize("kind,rows,dead", [("tracker", 1, 0), ("tracker", 1, 1), ("tracker", 2, 1), ("tracker", 64, 20), ("odd", 1024, 512),
                                            ("odd", 1025, 1000), ("tracker", 4100, 1300), ("long", 11, 5), ("odd", 9000, 0), ("odd", 9000, 9000),
                                            ("odd", 70001, 23456), ("odd", 131072, 40000), ("odd", 140001, 70000), ("odd", 131073, 131073),
                                            ("odd", 262144, 5), ("odd", 262145, 262140), ("odd", 300003, 123456), ("tracker", 17, 16)])
@pytest.mark.parametrize("offset", [0, 3])
def test_compact(kind, rows, dead, offset):
    """offset: of the flags from an aligned address."""
    bufs = buffers(kind, rows)
    want = host(bufs)
    g = torch.Generator().manual_seed(dead)
    mirror = torch.ones(rows, dtype=torch.bool)
    mirror[torch.randperm(rows, generator=g)[:dead]] = False
    c = int(mirror.sum())
    holes, movers = (~mirror[:c]).nonzero()[:, 0], mirror[c:].nonzero()[:, 0] + c
    now = torch.where(mirror, torch.arange(rows), torch.tensor(-1))
    now[movers] = holes
    for w in want:
        w[holes] = w[movers]
    flags = torch.ones(rows + 32, dtype=torch.bool, device="cuda")
    live = flags[offset:offset + rows]
    live.copy_(mirror)
    got, count = _rc().compact_rows(bufs, live)
    assert bool(flags[:offset].all()) and bool(flags[offset + rows:].all())
    assert count.tolist() == [c] and torch.equal(got.cpu(), now) and same(bufs, want)
    assert torch.equal(live.cpu(), torch.arange(rows) < c)


def test_empty_calls_and_an_empty_cache():
    rc = _rc()
    bufs = buffers("tracker", 4)
    want = host(bufs)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    live = torch.ones(4, dtype=torch.bool, device="cuda")
    rc.copy_rows(bufs, none, none)
    rc.free_rows(live, none)
    assert rc.fork_rows(bufs, live, none).shape == (0,) and same(bufs, want) and bool(live.all())
    empty = [torch.empty(0, 3, device="cuda")]
    now, count = rc.compact_rows(empty, torch.empty(0, dtype=torch.bool, device="cuda"))
    assert now.shape == (0,) and count.tolist() == [0]


@pytest.mark.parametrize("n", [1, 256, 257, 3000, 1 << 14, (1 << 14) + 1, 40000])
def test_copies_into_an_empty_cache(n):
    """No row number is good: nothing happens but the status bit, in all three forms of the copy."""
    g = torch.Generator().manual_seed(n)
    src, dst = torch.randint(-3, 9, (n,), generator=g).cuda(), torch.randint(-3, 9, (n,), generator=g).cuda()
    st = status()
    _rc().copy_rows([torch.empty(0, 3, device="cuda"), torch.empty(0, 2, 5, dtype=torch.uint8, device="cuda")], src, dst, st)
    assert int(st) == nat.STATUS_BAD_ROW


def test_rows_past_32_bits():
    """A row of 640 MB: the fourth starts past 2^31 bytes."""
    rows, n = 5, 160_000_000
    big = torch.zeros(rows, n, device="cuda")
    big[:, 0] = torch.arange(rows, device="cuda")
    big[:, -1] = torch.arange(rows, device="cuda") + 10
    _rc().copy_rows([big], torch.tensor([4, 3], device="cuda"), torch.tensor([3, 0], device="cuda"))
    assert big[:, 0].tolist() == [3, 1, 2, 4, 4] and big[:, -1].tolist() == [13, 11, 12, 14, 14]


def test_graph_replays():
    """free -> fork -> compact captured once and replayed on other contents; the sources and the freed rows come from memory."""
    rc = _rc()
    rows = 300
    bufs = buffers("tracker", rows)
    live = torch.ones(rows, dtype=torch.bool, device="cuda")
    drop, src = torch.zeros(7, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    src += 1
    for _ in range(2):
        rc.free_rows(live, drop)
        rc.fork_rows(bufs, live, src)
        rc.compact_rows(bufs, live)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rc.free_rows(live, drop)
        ids = rc.fork_rows(bufs, live, src)
        now, count = rc.compact_rows(bufs, live)
        rc.copy_rows(bufs, torch.stack([src[0], src[1]]), torch.stack([src[1], src[0]]))
    for k in range(4):
        fresh = buffers("tracker", rows, 50 + k)
        for b, f in zip(bufs, fresh):
            b.copy_(f)
        live.fill_(True)
        drop.copy_(torch.randperm(rows - 10, generator=torch.Generator().manual_seed(k))[:7] + 5)
        src.copy_(torch.tensor([0, 1, 2]))
        l2 = live.clone()
        graph.replay()
        rc.free_rows(l2, drop)
        i2 = rc.fork_rows(fresh, l2, src)
        n2, c2 = rc.compact_rows(fresh, l2)
        rc.copy_rows(fresh, torch.stack([src[0], src[1]]), torch.stack([src[1], src[0]]))
        torch.cuda.synchronize()
        assert torch.equal(ids, i2) and torch.equal(now, n2) and torch.equal(count, c2) and torch.equal(live, l2)
        assert all(torch.equal(a, b) for a, b in zip(bufs, fresh))


def test_what_a_call_writes_in_place_autograd_sees():
    """A tensor that a graph has saved and a call then overwrites: its backward pass raises, as after torch's own operations in
    place, instead of using the new content."""
    from umetrack_amd.lib.common import gated_filter as gf
    rc, one = _rc(), torch.tensor([1], device="cuda")

    def saved(t):
        w = torch.ones(1, device="cuda", requires_grad=True)
        return (t * w).sum()
    x, gate, live = torch.rand(2, 3, device="cuda"), torch.zeros(2, device="cuda"), torch.tensor([True, True, False], device="cuda")
    calls = {"out": lambda s: gf.gated_step(x, gate, torch.zeros(3, 3, device="cuda"), out=s[:2]), "state": lambda s: gf.gated_step(x, gate, s),
             "copy": lambda s: rc.copy_rows([s], one, one - 1), "fork": lambda s: rc.fork_rows([s], live.clone(), one),
             "compact": lambda s: rc.compact_rows([s], live.clone())}
    for name, call in calls.items():
        s = torch.rand(3, 3, device="cuda")
        loss = saved(s)
        call(s)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    for call in (lambda: rc.free_rows(live, one), lambda: rc.fork_rows([x.new_zeros(3, 1)], live, one), lambda: rc.compact_rows([x.new_zeros(3, 1)], live)):
        before = live._version
        call()
        assert live._version > before
    with pytest.raises(nat.UmtError, match="not differentiable"):
        gf.gated_step(x, gate, torch.zeros(3, 3, device="cuda"), out=torch.zeros(2, 3, device="cuda", requires_grad=True))
    read = x._version, gate._version
    gf.gated_step(x, gate, torch.zeros(3, 3, device="cuda"))
    gf.gated_scan(x[None], gate[None])
    assert (x._version, gate._version) == read
    with torch.inference_mode():
        s = torch.zeros(3, 3, device="cuda")
        gf.gated_step(x, gate, s)
        rc.copy_rows([s], one, one - 1)


def test_model_memory_moves_with_the_filter_state():
    """The model's temporal rows as one of the buffers: frames of two hands, the state of one hand forked, the other's row
    freed and the cache closed up; the fork then goes on exactly as the original does."""
    from umetrack_amd import arch
    from umetrack_amd.lib.models.model_loader import model_from_state_dict
    rc = _rc()
    m = model_from_state_dict(arch.make_synthetic_state(5)).to("cuda")
    g = torch.Generator().manual_seed(0)
    fused = [torch.randn(3, 72, 6, 6, generator=g).cuda() for _ in range(2)]
    cam0 = torch.eye(4).repeat(3, 1, 1).cuda()
    m.temporal_step(fused[0], cam0, torch.arange(3, device="cuda"), torch.zeros(3, dtype=torch.bool, device="cuda"), required_rows=3)
    m.reserve_memory(6)
    state = torch.randn(6, 21, 3, generator=g).cuda()
    before, sb = m.memory_state(), state.clone()
    live = torch.tensor([1, 1, 1, 0, 0, 0], dtype=torch.bool, device="cuda")
    rc.free_rows(live, torch.tensor([0], device="cuda"))
    ids = rc.fork_rows([m, state], live, torch.tensor([2, 1], device="cuda"))
    assert ids.tolist() == [0, 3]
    rc.free_rows(live, torch.tensor([1], device="cuda"))
    now, count = rc.compact_rows([m, state], live)
    assert now.tolist() == [0, -1, 2, 1, -1, -1] and count.tolist() == [3]
    after = m.memory_state()
    for r, o in ((0, 2), (1, 1), (2, 2)):
        assert all(torch.equal(a[r], b[o]) for a, b in zip(after, before)) and torch.equal(state[r], sb[o])
    f = torch.stack([fused[1][0], fused[1][1], fused[1][0]])
    out = m.temporal_step(f, cam0, torch.arange(3, device="cuda"), torch.ones(3, dtype=torch.bool, device="cuda"), required_rows=6)
    assert torch.equal(out[0], out[2])
    rc.copy_rows([m], torch.tensor([0, 2], device="cuda"), torch.tensor([2, 5], device="cuda"))
    assert np.array_equal(m.memory_state()[0][5].cpu().numpy(), m.memory_state()[0][2].cpu().numpy())
    m.check_status()
