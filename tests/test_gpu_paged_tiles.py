"""The attention over pages where each tile has a workgroup of its own, where one plan holds up to 2000 slots, and where q has
many more rows than the step's tokens need."""
import random

import pytest
import torch

from mkx.paged import page_attend

from _paged_ref import HALF, attend_ref, sees
from test_gpu_paged import BF, DEV, FP, Att, _near

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)


def _takes_tiles(t, max_q=None):
    """Whether the call has a workgroup for each tile: more than 2048 tiles, or two of 256 rows for each CU and more."""
    T, NQ = t.q.shape[:2]
    NK = t.kp.shape[2]
    G = NQ // NK
    rows = (T if max_q is None else min(max_q, T)) * G
    bm = 64 if rows <= 64 else 128 if rows <= 128 else 256
    tiles = T * G // bm + len(t.nq)
    return tiles > 2048 or (bm == 256 and tiles * NK >= 2 * torch.cuda.get_device_properties(0).multi_processor_count)


def _check_in_parts(t, out, part, some, rng, window=0, sinks=0, causal=True, max_q=None):
    """Some slots against the formula; all of them against calls of `part` slots each: either result is within about u of mean |v|
    for the probabilities' rounding and u of |o| for its own, 2 u max |v| together, and 32-bit sums are far below a sixteenth of it."""
    kw = dict(window=window, sinks=sinks, causal=causal)
    B, oc = len(t.nq), out.cpu()
    for b in some + rng.sample(range(B), 60):
        lo, hi = t.cu_l[b], t.cu_l[b + 1]
        o, tol = attend_ref(t.q[lo:hi], t.k[b], t.v[b], causal, window, sinks, t.q.shape[2] ** -0.5)
        _near(oc[lo:hi], o, tol, f"slot {b}: {t.nq[b]} of {t.n[b]}")
    top = max(float(v.double().abs().max()) for v in t.v if v.numel())
    want = torch.empty_like(out)
    for b in range(0, B, part):
        e = min(b + part, B)
        page_attend(t.qd, t.kp, t.vp, t.table[b:e], t.cu[b: e + 1].contiguous(), t.kv[b:e].contiguous(), max_q=max_q, out=want, **kw)
    lo, hi = t.cu_l[0], t.cu_l[-1]
    assert float((out[lo:hi].double() - want[lo:hi].double()).abs().max()) <= 4 * HALF[t.dt] * (1 + 2.0 ** -4) * top


@pytest.mark.parametrize("HD,dt", [(64, BF), (64, FP), (128, BF), (128, FP)])
@pytest.mark.parametrize("G,max_q", [(1, 2), (8, 2), (8, 16), (8, None)])
def test_attention_of_2048_slots(HD, dt, G, max_q):
    """Chunks of no, one and two tokens over caches of none and some, rows ahead of the first and behind the last: tiles of 64,
    128 and 256 rows."""
    rng = random.Random(HD + G)
    nq = [rng.choice([0, 1, 2]) for _ in range(2048)]
    nq[0], nq[1023], nq[2047] = 0, 2, 1
    n = [rng.choice([0, 1, a, a, a + 3, rng.randint(0, 40)]) for a in nq]
    n[5], n[2046] = 400, 270
    t = Att(nq, n, G, 1, HD, 16, dt, seed=G, lead=5, tail=7)
    assert _takes_tiles(t, max_q)
    for kw in (dict(), dict(causal=False), dict(window=9, sinks=2)):
        out = torch.full_like(t.qd, 5.0)
        t.run(out=out, max_q=max_q, **kw)
        _check_in_parts(t, out, 512, [0, 5, 1023, 2046, 2047], rng, max_q=max_q, **kw)
        assert bool((out[:5] == 5).all()) and bool((out[-7:] == 5).all())


@pytest.mark.parametrize("B", [513, 1025, 1537, 1900])
@pytest.mark.parametrize("HD,dt", [(64, FP), (128, BF)])
def test_attention_plans_of_many_slots(B, HD, dt):
    """One plan for all requests: two, three and four requests a thread, of one tile each and of several."""
    rng = random.Random(B)
    nq = [rng.choice([0, 1, 1, 1, 1, 1, 2]) for _ in range(B)]
    nq[3] = nq[B // 2] = nq[B - 2] = 33
    n = [rng.choice([a, a, a + 2, rng.randint(0, 30)]) for a in nq]
    n[7], n[B - 1] = 700, 300
    t = Att(nq, n, 2, 1, HD, 16, dt, seed=B, lead=1, tail=2)
    for max_q in (32, 33):  # a tile of 64 rows is not enough for the longest, or of 128 is
        assert not _takes_tiles(t, max_q)
        for kw in (dict(), dict(window=6, sinks=1)):
            _check_in_parts(t, t.run(max_q=max_q, **kw), 50, [3, 7, B // 2, B - 2, B - 1], rng, max_q=max_q, **kw)


@pytest.mark.parametrize("HD,dt,G", [(128, BF, 8), (128, FP, 4), (64, FP, 8)])
def test_attention_values_that_only_some_rows_see_by_tiles(HD, dt, G):
    """Infinities and NaN with a workgroup for each tile: in the rows that see them and in no others."""
    NK, B = 8, 70
    rng = random.Random(G)
    nq = [rng.choice([0, 1, 30, 70, 2]) for _ in range(B)]
    n = [a + rng.choice([0, 3, 100, -a]) for a in nq]
    nq[3], n[3], nq[9], n[9] = 300, 500, 90, 333
    t = Att(nq, n, NK * G, NK, HD, 16, dt, seed=G)
    assert _takes_tiles(t)
    inf, nan = float("inf"), float("nan")
    for b, j, h, d, x in ((3, 490, 0, 3, nan), (3, 470, 1, 60, inf), (3, 300, 7, 8, -inf), (9, 0, 0, 1, inf), (9, 250, 1, 17, nan), (9, 332, 5, 63, -inf),
                          (9, 300, 5, 63, inf), (3, 2, 0, 9, inf)):
        t.v[b][j, h, d] = x
        t.vp[t.table_l[b][j // 16], j % 16, h, d] = x
    for window, sinks in ((0, 0), (37, 5)):
        out = t.run(window=window, sinks=sinks).double().cpu()
        for b, q in enumerate(nq):
            o, tol = attend_ref(t.q[t.cu_l[b]: t.cu_l[b + 1]], t.k[b], torch.where(torch.isfinite(t.v[b]), t.v[b], 0), True, window, sinks, HD ** -0.5)
            for j, h, d in (~torch.isfinite(t.v[b])).nonzero().tolist():
                for i in range(q):
                    if sees(n[b] - q + i, j, n[b], True, window, sinks):
                        o[i, h * G: (h + 1) * G, d] += t.v[b][j, h, d].double()
            got, fin = out[t.cu_l[b]: t.cu_l[b + 1]], torch.isfinite(o)
            assert torch.equal(torch.isnan(got), torch.isnan(o)) and torch.equal(got[~fin & ~torch.isnan(o)], o[~fin & ~torch.isnan(o)]), b
            _near(got[fin], o[fin], tol[fin], f"slot {b}")


@pytest.mark.parametrize("HD,dt", [(128, BF), (64, FP)])
def test_attention_by_tiles_of_broken_lengths(HD, dt):
    """Lengths beyond the table and below 0, a cu that falls and leaves q: finite results, rows behind T untouched."""
    t = Att([3, 0, 40] + [1] * 2045, [60, 0, 90] + [5] * 2045, 8, 1, HD, 16, dt)
    assert _takes_tiles(t)
    t.kp.copy_(torch.nan_to_num(t.kp)), t.vp.copy_(torch.nan_to_num(t.vp))
    T = t.q.shape[0]
    whole = torch.full((T + 8, 8, HD), 3.0, dtype=dt, device=DEV)
    kv = t.kv.clone()
    kv[0], kv[1], kv[5] = 2 ** 31 - 1, -4, -2 ** 31
    cu = t.cu.clone()
    cu[10], cu[700], cu[900], cu[2048] = -3, 2 ** 31 - 1, 0, 2 ** 31 - 1
    table = t.table.clone()
    table[3, 0], table[4, 0] = 10 ** 6, -9
    page_attend(t.qd, t.kp, t.vp, table, cu, kv, out=whole[:T])
    assert bool((whole[T:] == 3).all()) and bool(torch.isfinite(whole).all())
    whole[:T] = 3
    page_attend(t.qd, t.kp, t.vp, table, t.cu, kv, out=whole[:T])
    assert bool((whole[t.cu_l[3]: t.cu_l[5]] == 0).all()) and bool((whole[t.cu_l[5]: t.cu_l[6]] == 0).all())


@pytest.mark.parametrize("max_q", [1, 5, 333, None])
@pytest.mark.parametrize("B,T", [(64, 16384), (24, 9000)])
def test_attention_of_a_padded_step(B, T, max_q):
    """A step of few tokens in a q of a captured step's capacity, with bounds that are right, too high and too low: the rows decide
    which kernel runs, and nothing else depends on it."""
    rng = random.Random(B)
    nq = [rng.choice([0, 1, 1, 1]) for _ in range(B)]
    nq[1], nq[2] = 1, 7
    n = [a + rng.randint(0, 300) for a in nq]
    n[1] = 3000
    t = Att(nq, n, 16, 2, 128, 64, BF, seed=B, tail=T - sum(nq))
    out = torch.full_like(t.qd, 5.0)
    t.run(out=out, max_q=max_q, window=256, sinks=4)
    t.check(out, window=256, sinks=4)
    assert bool((out[t.cu_l[-1]:] == 5).all())
    t.check(t.run(out=out, max_q=max_q))
    assert torch.equal(t.run(max_q=max_q)[: t.cu_l[-1]], out[: t.cu_l[-1]])
