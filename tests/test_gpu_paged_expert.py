"""From the paged cache to the expert: prompts and frames are stored and attended step by step, their projected results are the
context whose source caches the expert reads."""
from dataclasses import replace

import pytest
import torch

from _cases import TINY, diff, make_case, oracle_dims, oracle_steps
from _paged_ref import HALF, attend_ref, rope_ref
from mkx import ExpertMegakernel, synthetic as SY
from mkx.paged import AxesRotary, PagedCache
from mkx.prepare import SourcePrepare
from oracle import expert_ref as ER

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)


def test_context_of_paged_tokens_reaches_the_expert():
    B, NQ, NK, HD, cap = 3, 4, 2, 64, 64
    steps = [[20, 7, 30], [15, 1, 0]]
    lens = [sum(s) for s in zip(*steps)]
    cfg = replace(TINY, B=B)
    case = make_case(cfg, ca_len=lens)
    model, past = case["model"], case["past"]
    cache = PagedCache(1, NK, HD, 12, slots=B, table_cols=4, max_tokens=cap, page_rows=16)
    axis = AxesRotary.sections((16, 16))
    rope = AxesRotary(HD, axis)
    prep = SourcePrepare(model)
    g = torch.Generator().manual_seed(6)
    w_out = (torch.randn(cfg.ctx_dim, NQ * HD, generator=g) * (NQ * HD) ** -0.5).cuda()
    context = torch.zeros(B, cfg.SP, cfg.ctx_dim, device="cuda")
    kept = [([], [], []) for _ in range(B)]
    freqs = 10000.0 ** (-torch.arange(0, HD, 2, dtype=torch.float64) / HD)
    for add in steps:
        n = sum(add)
        x = torch.randn(n, NQ + 2 * NK, HD, generator=g).to(torch.bfloat16)
        pos = torch.randint(0, 40, (2, n), generator=g, dtype=torch.int32)
        q, k, v = x.cuda().split([NQ, NK, NK], 1)
        m = cache.append(torch.tensor(add, dtype=torch.int32, device="cuda"))
        q = cache.store(0, rope, q, k, v, pos.cuda(), m)
        o = cache.attend(0, q, m, max_q=max(add), causal=False)
        slot = torch.searchsorted(m.cu, torch.arange(n, dtype=torch.int32, device="cuda"), right=True) - 1
        context[slot, m.pos[:n].long()] = o.flatten(1).float() @ w_out.t()
        for b in range(B):
            lo, hi = m.cu[b].item(), m.cu[b + 1].item()
            kx, vx, rows = kept[b]
            if hi == lo:
                continue
            kx.append(rope_ref(x[lo:hi, NQ: NQ + NK], pos[:, lo:hi], axis, freqs)[0].to(torch.bfloat16))
            vx.append(x[lo:hi, NQ + NK:])
            want, tol = attend_ref(q[lo:hi].cpu(), torch.cat(kx), torch.cat(vx), False, 0, 0, HD ** -0.5)
            # a stored key's element may round to its other neighbour where the 32-bit turn lies next to the border, a step of 2 u:
            # a score moves by at most 2 u |q| . |k|, every probability by that much relative, on both sides of the quotient
            move = 2 * HALF[torch.bfloat16] * float((q[lo:hi].double().cpu().norm(dim=-1).max()) * torch.cat(kx).double().norm(dim=-1).max()) * HD ** -0.5
            tol = tol + 2 * move * torch.cat(vx).double().abs().max()
            w = w_out.double().cpu()
            # 256 products in 32 bits: 2^-24 each of what is summed so far
            err = tol.flatten(1) @ w.abs().t() + 2.0 ** -16 * (want.abs() + tol).flatten(1) @ w.abs().t()
            off = (context[b, m.kv_len[b].item() - (hi - lo): m.kv_len[b].item()].double().cpu() - want.flatten(1) @ w.t()).abs()
            assert bool((off <= err).all()), (b, float((off - err).max()))
    assert m.kv_len.tolist() == lens
    past.cross_attn_kv = prep(context, m.kv_len)
    # SourcePrepare reads the context in bf16
    ref = ER.register_prepare(context.to(torch.bfloat16).float().cpu(), lens, case["inp"]["mem_states"][:, :0], [0] * B, SY.oracle_weights(case["W"]), oracle_dims(cfg), cfg.m_q,
                              mode="mirror")
    for i, name in enumerate(("kca", "vca")):
        got = torch.stack([kv[i] for kv in past.cross_attn_kv]).float().cpu()
        r = ref[name].float()
        bound = 2.0 ** -6 * torch.sqrt(r[..., :32] ** 2 + r[..., 32:] ** 2).repeat(1, 1, 1, 1, 2) + 1e-6 if i == 0 else 2.0 ** -7 * r.abs() + 2.0 ** -12
        assert bool(((got - r).abs() <= bound).all()), name
        for b in range(B):
            assert bool((got[:, b, lens[b]:] == 0).all())
    mk = ExpertMegakernel(model)
    x1, _, _ = model._expert_first_step(case["noise"], past, None, case["mods"][..., :1, :], case["dt"], cfg.action_dim)
    x = mk.run(x1, case["mods"], case["dt"], past, cfg.action_dim)
    mk.check()
    torch.cuda.synchronize()
    worst, mean = diff(x, oracle_steps(case, x1, 1, cfg.num_steps - 1, "fp32"), cfg.action_dim)
    assert worst <= 1e-3 and mean <= 2e-4
