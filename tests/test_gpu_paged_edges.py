"""The paged cache's operators in calls beside the ordinary ones: requests that were not granted, positions and weights of other
types, sizes at the launch's limits, the attention's other kernel."""
import math
import random
from fractions import Fraction

import pytest
import torch

from mkx import _lib
from mkx.paged import AxesRotary, PagedCache, PagePool, page_attend

from _paged_ref import HALF, attend_ref, map_ref, rope_ref, sees
from test_gpu_paged import BF, DEV, FP, Att, _near, i32

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)


# ---- requests that were not granted -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("how", [dict(), dict(max_q=40), dict(causal=False), dict(window=20, sinks=3)])
@pytest.mark.parametrize("graph", [False, True])
def test_rows_of_refused_requests_are_zero(how, graph):
    """Steps whose pool or whose table row runs out: the refused requests' rows are zeros, the others' their attention, and
    rows behind the tokens stay; a request refused once is served when its pages are there."""
    NQ, NK, HD, B, P, cap = 4, 2, 64, 5, 16, 120
    cache = PagedCache(1, NK, HD, 9, slots=B, table_cols=4, max_tokens=cap, page_rows=P, device=DEV)
    for t in cache.k + cache.v:
        t.fill_(float("nan"))
    rope = AxesRotary(HD, [0] * (HD // 2), device=DEV)
    add, done = i32([0] * B), i32([0] * B)
    g = torch.Generator().manual_seed(3)
    x, pos = torch.zeros(cap, NQ + 2 * NK, HD, dtype=BF, device=DEV), torch.arange(cap, dtype=torch.int32, device=DEV)
    out = torch.zeros(cap, NQ, HD, dtype=BF, device=DEV)
    q = torch.zeros(cap, NQ, HD, dtype=BF, device=DEV)

    def step():
        m = cache.append(add, done)
        a, k, v = x.split([NQ, NK, NK], 1)
        cache.store(0, rope, a, k, v, pos, m, q_out=q)
        cache.attend(0, q, m, out=out, **how)
        return m

    graphs, maps = [], []
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(), step()
        torch.cuda.current_stream().wait_stream(side)
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                maps.append(step())
            graphs.append(gr)
    # 9 pages of 16: 30 + 20 + 1 + 0 + 40 tokens take 2 + 2 + 1 + 0 + 3; slot 0 then wants 2 more, one too many, slot 2 more than its
    # table row; slot 1 ends, and slot 0 has its pages
    steps = [([30, 20, 1, 0, 40], [0] * 5, [1, 1, 1, 1, 1]), ([33, 5, 1, 0, 2], [0] * 5, [0, 1, 1, 1, 1]),
             ([0, 0, 64, 0, 1], [0, 1, 0, 0, 0], [1, 0, 0, 1, 1]), ([33, 3, 1, 0, 1], [0] * 5, [1, 1, 1, 1, 1])]
    for i, (a, d, granted) in enumerate(steps):
        add.copy_(i32(a)), done.copy_(i32(d))
        x.copy_(torch.randn(x.shape, generator=g).to(BF))
        out.fill_(9.0)
        if graph:
            graphs[i % 2].replay()
            m = maps[i % 2]
        else:
            m = step()
        torch.cuda.synchronize()
        assert m.granted.tolist() == granted, i
        cu, n, table = m.cu.tolist(), m.kv_len.tolist(), m.table.tolist()
        got, qc = out.cpu(), q.cpu()
        assert bool((got[cu[-1]:] == 9).all())
        for b in range(B):
            lo, hi = cu[b], cu[b + 1]
            if not granted[b]:
                assert bool((got[lo:hi] == 0).all()), (i, b)
                continue
            held = table[b][: -(-n[b] // P)]
            k, v = (t[0][held].flatten(0, 1)[: n[b]].cpu() for t in (cache.k, cache.v))
            o, tol = attend_ref(qc[lo:hi], k, v, how.get("causal", True), how.get("window", 0), how.get("sinks", 0), HD ** -0.5)
            _near(got[lo:hi], o, tol, (i, b))


@pytest.mark.parametrize("max_q,B", [(1, 3), (None, 3), (None, 70), (None, 2048)])
def test_attention_of_some_granted_requests(max_q, B):
    """Every plan: requests in a wave's registers, tiles in them, a workgroup's plan, a workgroup for each tile."""
    rng = random.Random(B)
    nq = [rng.choice([1, 2, 0, 70 if B == 3 else 3]) for _ in range(B)]
    nq[0] = 1
    n = [x + rng.choice([0, 5, 40]) for x in nq]
    t = Att(nq, n, 8, 1, 64, 16, FP, seed=B, lead=2, tail=3)
    granted = [rng.choice([0, 1, -5]) for _ in range(B)]
    granted[-1] = 0
    out = torch.full_like(t.qd, 7.0)
    t.run(out=out, max_q=max_q, granted=i32(granted))
    full = t.run(max_q=max_q)
    for b in range(B):
        lo, hi = t.cu_l[b], t.cu_l[b + 1]
        assert torch.equal(out[lo:hi], full[lo:hi] if granted[b] else torch.zeros_like(full[lo:hi])), b
    assert bool((out[:2] == 7).all()) and bool((out[-3:] == 7).all())
    with pytest.raises(ValueError, match="granted"):
        t.run(granted=i32(granted + [1]))
    with pytest.raises(ValueError, match="granted"):
        t.run(granted=i32(granted).long())
    with pytest.raises(ValueError, match="granted is on cpu"):
        t.run(granted=torch.ones(B, dtype=torch.int32))


# ---- launches of the largest sizes ------------------------------------------------------------------------------------------------

def test_rope_of_more_tokens_than_a_launch_has_workgroups():
    """2^24 workgroups of 256 threads are one more than a launch takes; 33 heads of 64, stored, are a token each."""
    HD, NK, T, P = 64, 33, (1 << 24) + 70, 16
    at = [0, 1, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, T - 1]
    rope = AxesRotary(HD, AxesRotary.sections((16, 16)), q_norm=torch.zeros(HD, device=DEV, dtype=BF), device=DEV)
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v = (torch.randn(1, n, HD, generator=g, device=DEV).to(BF) for n in (1, NK, NK))
    pos = torch.stack([torch.arange(T, device=DEV), T - torch.arange(T, device=DEV)])
    slots = torch.full((T,), -1, dtype=torch.int64, device=DEV)
    slots[at] = torch.arange(len(at), device=DEV) + 3
    for positions in (pos.int(), pos):
        kp, vp = (torch.zeros(2, P, NK, HD, dtype=BF, device=DEV) for _ in range(2))
        out = torch.full((T + 1, 1, HD), 9.0, dtype=BF, device=DEV)
        rope.store(q.expand(T, 1, HD), k.expand(T, NK, HD), v.expand(T, NK, HD), positions, kp, vp, slots, q_out=out[:T])
        n = len(at)
        kw, vw = torch.zeros_like(kp), torch.zeros_like(vp)
        want = rope.store(q.expand(n, 1, HD), k.expand(n, NK, HD), v.expand(n, NK, HD), positions[:, at].contiguous(), kw, vw, slots[at])
        assert torch.equal(out[at], want) and torch.equal(kp, kw) and torch.equal(vp, vw)
        assert bool((out[T] == 9).all()) and bool((out[:T].view(torch.int16) != out[T, 0, 0].view(torch.int16)).any(-1).all())


@pytest.mark.parametrize("lead", [0, 1 << 28, 1 << 29])
def test_attention_of_more_rows_than_a_launch_has_workgroups_for(lead):
    """A q of 2^29 rows, nearly all of them no request's, with max_q = 1: tiles of 64 rows would be 2^23 workgroups of 512."""
    t = Att([1, 1, 1], [300, 5, 70], 1, 1, 64, 16, BF, seed=2)
    T = (1 << 29) + 100
    t.q[:] = t.q[:1].clone()
    out = torch.empty(T, 1, 64, dtype=BF, device=DEV)  # 64 GiB, nearly none of them touched
    out[lead: lead + 9] = 4.0
    page_attend(t.qd[:1].expand(T, 1, 64), t.kp, t.vp, t.table, t.cu + lead, t.kv, max_q=1, out=out)
    t.check(out[lead: lead + 3])
    assert bool((out[lead + 3: lead + 9] == 4).all())
    del out
    torch.cuda.empty_cache()


# ---- rotary: positions and weights as they are given ----------------------------------------------------------------------------

def _far_turns(rope, pos, hd):
    """(cos, sin) [T, 1, hd / 2] of positions of any size: the turns' fractions as whole numbers give them, in 64 bits after that."""
    turns, axis = [Fraction(x) for x in rope._turns.tolist()], rope._axis.tolist()
    frac = torch.tensor([[float(Fraction(int(pos[a, t])) * turns[i] % 1) for i, a in enumerate(axis)] for t in range(pos.shape[1])], dtype=torch.float64)
    ang = 2 * math.pi * frac[:, None]
    return torch.cos(ang), torch.sin(ang)


@pytest.mark.parametrize("layout", ["plain", "strided", "one_axis"])
@pytest.mark.parametrize("store", [False, True])
def test_rope_positions_beyond_32_bits(layout, store):
    """64-bit positions turn by their own angle, whatever their upper half holds."""
    HD, T, axes = 64, 40, 1 if layout == "one_axis" else 3
    g = torch.Generator().manual_seed(5)
    rope = AxesRotary(HD, [0] * 32 if axes == 1 else AxesRotary.sections((10, 11, 11)), device=DEV)
    pos = torch.randint(-(1 << 44), 1 << 44, (axes, T), generator=g)
    pos[:, :8] = torch.tensor([0, -1, (1 << 31) - 1, 1 << 31, -(1 << 31), (1 << 32) + 3, 1 << 52, -(1 << 40) - 7])
    posd = pos.to(DEV)
    if layout == "strided":
        posd = torch.stack([posd, posd + 1], -1).flatten(1)[:, ::2]
        assert posd.stride(1) == 2
    elif layout == "one_axis":
        posd = posd[0]
    x = torch.randn(T, 3, HD, generator=g).to(BF)
    xd = x.to(DEV)
    if store:
        kp, vp = (torch.zeros(3, 16, 3, HD, dtype=BF, device=DEV) for _ in range(2))
        rope.store(None, xd, xd, posd, kp, vp, torch.arange(T, device=DEV))
        got = kp.view(-1, 3, HD)[:T]
    else:
        got = rope(xd, None, posd)[0]
    c, s = _far_turns(rope, pos, HD)
    lo, hi = x[..., :32].double(), x[..., 32:].double()
    want = torch.cat([lo * c - hi * s, hi * c + lo * s], -1)
    # as in rope_ref: the fraction of a turn, its sine and cosine and the products in 32 bits; the product of position and turns
    # is exact up to 2^-53 of its own rounding's size
    mix = lo.abs() + hi.abs()
    _near(got, want, HALF[BF] * want.abs() * (1 + 2.0 ** -8) + 2.0 ** -20 * torch.cat([mix, mix], -1))


@pytest.mark.parametrize("HD,dt,wt", [(64, BF, torch.float32), (128, FP, torch.float32), (128, BF, torch.float64), (64, BF, FP), (128, FP, BF)])
def test_rope_norm_weights_of_other_types(HD, dt, wt):
    """Weights of more bits than the tokens, or of the other 16-bit type, are not rounded to the tokens' type: plain weights near
    0.1, passed as w - 1, keep their place."""
    g = torch.Generator().manual_seed(9)
    T = 37
    plain = 0.1 + 0.01 * torch.randn(HD, generator=g, dtype=torch.float64)
    wq, wk = ((plain - 1).to(wt), (torch.randn(HD, generator=g) * 1e-3).to(wt))
    rope = AxesRotary(HD, [0] * (HD // 2), q_norm=wq.to(DEV), k_norm=wk.to(DEV), eps=1e-5, device=DEV)
    x = torch.randn(T, 5, HD, generator=g).to(dt)
    pos = torch.arange(T, dtype=torch.int32)[None]
    freqs = 10000.0 ** (-torch.arange(0, HD, 2, dtype=torch.float64) / HD)
    q, k = rope(x[:, :3].to(DEV), x[:, 3:].to(DEV), pos.to(DEV))
    for got, part, w in ((q, x[:, :3], wq), (k, x[:, 3:], wk)):
        want, tol = rope_ref(part, pos, [0] * (HD // 2), freqs, w, 1e-5)
        # 1 + w in 32 bits: 2^-24 of the sum's 1, which is 2^-20 of a weight of 0.07 and more
        _near(got, want, tol)
    # one of them of the tokens' type, the other not
    rope = AxesRotary(HD, [0] * (HD // 2), q_norm=wq.to(DEV), k_norm=wk.to(dt).to(DEV), eps=1e-5, device=DEV)
    q2, k2 = rope(x[:, :3].to(DEV), x[:, 3:].to(DEV), pos.to(DEV))
    want, tol = rope_ref(x[:, 3:], pos, [0] * (HD // 2), freqs, wk.to(dt), 1e-5)
    _near(k2, want, tol)
    assert torch.equal(q2, q)
    both = AxesRotary(HD, [0] * (HD // 2), q_norm=wk.to(dt).to(DEV), k_norm=wk.to(dt).to(DEV), eps=1e-5, device=DEV)
    assert torch.equal(both(None, x[:, 3:].to(DEV), pos.to(DEV))[1], k2)


# ---- gradients ------------------------------------------------------------------------------------------------------------------

def test_inputs_that_require_grad_are_refused():
    """No operator here has a backward pass: an input that asks for one is refused aloud, and served under no_grad."""
    t = Att([3], [20], 4, 2, 64, 16, BF)
    rope = AxesRotary(64, [0] * 32, q_norm=torch.nn.Parameter(torch.zeros(64, device=DEV, dtype=BF)), device=DEV)
    x, pos = torch.randn(3, 2, 64, device=DEV).to(BF), torch.arange(3, dtype=torch.int32, device=DEV)
    slots = torch.arange(3, device=DEV)
    leaf = lambda y: y.clone().requires_grad_()  # noqa: E731
    calls = {"q": lambda: rope(leaf(x), x, pos), "k": lambda: rope(x, leaf(x), pos),
             "v": lambda: rope.store(x, x, leaf(x), pos, t.kp, t.vp, slots), "q_out": lambda: rope(x, None, pos, q_out=leaf(x)),
             "k_out": lambda: rope(None, x, pos, k_out=leaf(x)), "k_pages": lambda: rope.store(x, x, x, pos, leaf(t.kp), t.vp, slots),
             "v_pages": lambda: rope.store(x, x, x, pos, t.kp, leaf(t.vp), slots)}
    attend = lambda **kw: page_attend(*[kw.get(n, y) for n, y in (("q", t.qd), ("k_pages", t.kp), ("v_pages", t.vp))],  # noqa: E731
                                      t.table, t.cu, t.kv, out=kw.get("out"))
    more = {"q": lambda: attend(q=leaf(t.qd)), "k_pages": lambda: attend(k_pages=leaf(t.kp)), "v_pages": lambda: attend(v_pages=leaf(t.vp)),
            "out": lambda: attend(out=leaf(t.qd))}
    for name, call in [*calls.items(), *more.items()]:
        with torch.enable_grad(), pytest.raises(ValueError, match=f"^{name} requires grad"):
            call()
        with torch.no_grad():
            call()
    with torch.enable_grad():  # a weight may, it was copied
        assert not rope(x, x, pos)[0].requires_grad and not attend().requires_grad
    with torch.inference_mode():
        rope(leaf(x), x, pos), attend()


# ---- outputs in their inputs' buffers ------------------------------------------------------------------------------------------


def test_outputs_beside_inputs_in_one_buffer():
    """Results that go between the heads of their inputs, or before and behind them, are no overlap."""
    g = torch.Generator().manual_seed(8)
    rope = AxesRotary(64, [0] * 32, device=DEV)
    x = torch.randn(40, 12, 64, generator=g).to(BF).to(DEV)
    pos = torch.arange(40, dtype=torch.int32, device=DEV)
    q, k = rope(x[:, :3], x[:, 6:9], pos)
    y = x.clone()
    rope(y[:, :3], y[:, 6:9], pos, q_out=y[:, 3:6], k_out=y[:, 9:])
    assert torch.equal(y[:, 3:6], q) and torch.equal(y[:, 9:], k) and torch.equal(y[:, :3], x[:, :3]) and torch.equal(y[:, 6:9], x[:, 6:9])
    for out in (y[:, 1:4], y[:, 5:8]):
        with pytest.raises(_lib.MkxError, match="shares elements"):
            rope(y[:, :3], y[:, 6:9], pos, q_out=out, k_out=y[:, 9:])
    t = Att([40], [40], 4, 2, 64, 16, BF)
    both = torch.zeros(41, 8, 64, dtype=BF, device=DEV)
    both[:40, :4] = t.qd
    assert torch.equal(page_attend(both[:40, :4], t.kp, t.vp, t.table, t.cu, t.kv, out=both[:40, 4:]), t.run())
    for out in (both[1:, :4], both[:40, 2:6]):
        with pytest.raises(_lib.MkxError, match="shares elements"):
            page_attend(both[:40, :4], t.kp, t.vp, t.table, t.cu, t.kv, out=out)


# ---- who waits for whom -----------------------------------------------------------------------------------------------------------

def test_map_refused_needs_hold_up_later_slots():
    """A prompt that lacks pages counts against the slots behind it: those that need a page are refused with it, those that need none
    are not; with add = 0 for the prompt they pass. Tokens count against max_tokens whether granted or not, pages that no table
    row holds against nobody."""
    P, cols, N, T = 16, 4, 6, 90
    pool = PagePool(4, N, P, cols, T, DEV)
    length, table, queue, head, free = [0] * 4, [[-1] * cols for _ in range(4)], list(range(N)), 0, N
    for add, granted in (([0, 16, 20, 0], [1, 1, 1, 1]),      # 3 pages taken, 3 free
                         ([50, 1, 1, 1], [0, 0, 1, 0]),       # 4 are too many; then 1 more each, though 3 are free; slot 2 needs none
                         ([0, 1, 1, 1], [1, 1, 1, 1]),        # 1 free
                         ([41, 1, 19, 0], [0, 1, 0, 1]),      # 3 pages, then 1 more; slot 1 needs none
                         ([75, 0, 1, 16], [0, 1, 1, 0]),      # more than a row holds; slot 3's tokens end behind T
                         ([65, 0, 0, 16], [0, 1, 1, 1])):     # the same, and slot 3 gets the last page
        want = map_ref(add, None, length, head, free, table, queue, P, T)
        assert want["granted"] == granted, add
        m = pool.append(i32(add))
        for name, w in want.items():
            assert getattr(m, name).tolist() == w, (add, name)
        length, table, queue, (head, free) = want["kv_len"], want["table"], want["queue"], want["ends"]


def test_pool_after_replays_of_both_graphs():
    """The pool's own view, a load and eager appends between replays: right after as many replays of the one graph as of the other."""
    P, cols, N, T, B = 16, 5, 12, 50, 3
    pool = PagePool(B, N, P, cols, T, DEV)
    add, done = i32([0] * B), i32([0] * B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        pool.append(add, done), pool.append(add, done)
    torch.cuda.current_stream().wait_stream(side)
    graphs, maps = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            maps.append(pool.append(add, done))
        graphs.append(gr)
    state = [0] * B, [[-1] * cols for _ in range(B)], list(range(N)), 0, N
    saved = None
    todo = [([9, 20, 0], "g"), ([9, 1, 16], "g"), ([1, 1, 1], "e"), ([0, 30, 1], "e"), ([2, 0, 1], "g"), ([-1, 3, 1], "g"), ([5, 5, 5], "e"), ([1, 0, 0], "e")]
    for i, (a, how) in enumerate(todo):
        ended = [0, 0, int(i == 3)]
        add.copy_(i32(a)), done.copy_(i32(ended))
        want = map_ref(a, ended, *state[:1], state[3], state[4], state[1], state[2], P, T)
        if how == "g":
            graphs[i % 2].replay()
            m = maps[i % 2]
        else:
            m = pool.append(add, done)
        for name, w in want.items():
            assert getattr(m, name).tolist() == w, (i, name)
        state = want["kv_len"], want["table"], want["queue"], *want["ends"]
        if i % 2:
            assert pool.kv_len.tolist() == state[0] and pool.ends.tolist() == list(state[3:])
            got = pool.state_dict()
            if i == 3:
                saved = got, state
    pool.load_state_dict(saved[0])
    state = saved[1]
    for i, a in enumerate(([4, 4, 4], [1, 1, 1])):
        add.copy_(i32(a)), done.zero_()
        want = map_ref(a, None, state[0], state[3], state[4], state[1], state[2], P, T)
        graphs[i].replay()
        for name, w in want.items():
            assert getattr(maps[i], name).tolist() == w, (i, name)
        state = want["kv_len"], want["table"], want["queue"], *want["ends"]


# ---- keys that are not numbers ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("HD,dt,G,NK,max_q", [(128, BF, 8, 2, 40), (64, FP, 1, 3, 40), (128, FP, 4, 40, None), (64, BF, 8, 1, 5)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_keys_that_only_some_rows_see(HD, dt, G, NK, max_q, bad):
    """NaN and infinite keys of the chunk itself and at the window's edge, under NaN queries of other tokens: the rows that see
    them are no numbers, the others what they are without."""
    nq, n, W, S = [40, 3, 1, 200], [300, 260, 77, 390], 37, 5
    t = Att(nq, n, NK * G, NK, HD, 16, dt, seed=G)
    spoilt = {(0, 290): 0, (0, 255): NK - 1, (1, 258): 0, (1, 2): 0, (3, 380): 0, (3, 388): NK - 1, (3, 120): 0}
    for (b, j), h in spoilt.items():
        t.k[b][j, h] = bad
        t.kp[t.table_l[b][j // 16], j % 16, h] = bad
    dead = {(0, 3), (3, 77), (3, 199)}  # these queries themselves
    for b, i in dead:
        t.q[t.cu_l[b] + i] = float("nan")
        t.qd[t.cu_l[b] + i] = float("nan")
    for window, sinks in ((0, 0), (W, S)):
        out = t.run(window=window, sinks=sinks, max_q=max_q).double().cpu()
        for b, q in enumerate(nq):
            live = t.q[t.cu_l[b]: t.cu_l[b + 1]].nan_to_num(0.0)
            o, tol = attend_ref(live, t.k[b].nan_to_num(0.0, 0.0, 0.0), t.v[b], True, window, sinks, HD ** -0.5)
            got = out[t.cu_l[b]: t.cu_l[b + 1]]
            no = torch.zeros(q, NK, dtype=torch.bool)
            for i in range(q):
                for (c, j), h in spoilt.items():
                    no[i, h] |= c == b and sees(n[b] - q + i, j, n[b], True, window, sinks)
                no[i] |= (b, i) in dead
            no = no.repeat_interleave(G, 1)
            if bad != bad:
                assert bool(torch.isnan(got[no]).all()), b
            _near(got[~no], o[~no], tol[~no], (b, window))
