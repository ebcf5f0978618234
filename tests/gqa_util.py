"""Plain 64-bit forms of the grouped-query cache operators and the inputs of their tests."""
from __future__ import annotations

import numpy as np
import torch

import cautreo_b200 as ct

QMAX = {ct.CT_KV_INT8: 127.0, ct.CT_KV_E4M3: 448.0}
BF16_HALF = 2.0 ** -8             # largest relative error of one rounding to bf16


def encode(x: np.ndarray, dtype):
    """Codes and scales of fp32 rows x [..., dim]: every operation a single rounding to 32 bits."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        top = np.abs(x).max(-1, keepdims=True)            # NaN propagates
        fine = np.isfinite(top)
        d = (top / np.float32(QMAX[dtype])).astype(np.float32)
        inv = np.where(d > 0, np.minimum(np.float32(1) / d, np.finfo(np.float32).max), np.float32(0)).astype(np.float32)
        y = np.where(fine, x, np.float32(0)) * np.where(fine, inv, np.float32(0))
        if dtype == ct.CT_KV_INT8:
            codes = np.clip(np.floor(y + np.float32(0.5)), -127, 127).astype(np.int8)
        else:
            codes = torch.from_numpy(np.clip(y, -448, 448)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    return codes, np.where(fine, d, np.float32(np.nan))[..., 0].astype(np.float32)


def values(codes: torch.Tensor, scales, dtype) -> torch.Tensor:
    """What stored rows stand for, in 64 bits."""
    if dtype == ct.CT_KV_BF16:
        return codes.double()
    x = codes.double() if dtype == ct.CT_KV_INT8 else codes.view(torch.float8_e4m3fn).double()
    return x * scales.double()[..., None]


def kv_head(h, hq, hkv, order):
    return h % hkv if order == ct.CT_GQA_MODULO else h * hkv // hq


def attend(q, pool, scales, table, lens, dtype, hq, order, window=0, pages=None, scale=None):
    """(out, lse, weight, slack) in 64 bits: weight = sum_t p_t |v_t|, slack = the largest scale * sum_d |q_d k_td| of a
    row, what the error of a 32-bit evaluation is measured by.  Lengths and tables as the kernels take them."""
    S = len(lens)
    NP, _, H, P, D = pool.shape
    MP = table.shape[1]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    out = torch.zeros(S, hq, D, dtype=torch.float64, device=pool.device)
    weight = torch.zeros_like(out)
    lse = torch.full((S, hq), -np.inf, dtype=torch.float64, device=pool.device)
    slack = torch.zeros(S, hq, dtype=torch.float64, device=pool.device)
    tb = table.cpu().numpy()
    for s, n in enumerate(lens):
        n = min(max(int(n), 0), MP * P)
        start = max(0, n - window) if window else 0
        for kv in range(H):
            lps = range(start // P, -(-n // P)) if pages is None else [int(x) for x in pages[s][kv]]
            at, pos = [], []
            for lp in lps:
                if not 0 <= lp < MP or not 0 <= tb[s, lp] < NP:
                    continue
                for t in range(max(start, lp * P), min(n, lp * P + P)):
                    at.append((tb[s, lp], t - lp * P))
            if not at:
                continue
            pg = torch.tensor([a[0] for a in at], device=pool.device)
            sl = torch.tensor([a[1] for a in at], device=pool.device)
            k = values(pool[pg, 0, kv, sl], None if scales is None else scales[pg, 0, kv, sl], dtype)
            v = values(pool[pg, 1, kv, sl], None if scales is None else scales[pg, 1, kv, sl], dtype)
            for h in range(hq):
                if kv_head(h, hq, H, order) != kv:
                    continue
                qh = q[s, h].double()
                x = (k @ qh) * scale
                top = x.max()
                p = torch.exp(x - top)
                tot = p.sum()
                out[s, h] = (p @ v) / tot
                weight[s, h] = (p @ v.abs()) / tot
                lse[s, h] = top + torch.log(tot)
                slack[s, h] = (k.abs() @ qh.abs()).max() * scale
    return out, lse, weight, slack


def check_attention(got, got_lse, ref, dim, n_tokens, dtype):
    """|out - want| <= one rounding to bf16 + e * sum p |v|, with e the error that 32-bit scores, the exponential and
    rounded weights leave: a score is off by at most (dim + 4) roundings of its largest partial sum, 2^-23 each
    (the products of bf16 values are exact), so each p by twice that relative to the sum; bf16 pools take p as two bf16
    digits, off by 2^-16; 8-bit pools take p times the V scale as one fp16 value, off by half a step, 2^-11 relative, so
    by 2^-11 sum p |v| in all (and by 2^-25 where it is below 2^-14, in a unit where the largest weight of a step is 2^7
    or more: 2^-32 n of that); the exponential and the sums of the parts are off by 2^-18; the sum over n tokens adds
    n / 16 accumulations of 2^-24 a warp, of values that may cancel, hence relative to sum p |v|."""
    out, lse, weight, slack = ref
    score = (dim + 4) * 2.0 ** -23 * slack
    e = 2 * score + 2.0 ** -15 + n_tokens / 16 * 2.0 ** -23
    if dtype != ct.CT_KV_BF16:
        e = e + 2.0 ** -11
    err = (got.double() - out).abs()
    bound = BF16_HALF * (out.abs() + e[..., None] * weight) + e[..., None] * weight + 1e-38
    assert (err <= bound).all(), float((err - bound).max())
    if got_lse is not None:
        fin = torch.isfinite(lse)
        assert torch.equal(fin, torch.isfinite(got_lse))
        assert torch.equal(lse[~fin], got_lse[~fin].double())
        d = (got_lse.double() - lse).abs()[fin]
        lim = (score + 2.0 ** -18 + n_tokens / 16 * 2.0 ** -23)[fin] + 2.0 ** -22 * lse[fin].abs()
        assert (d <= lim).all(), float((d - lim).max())


def make_pool(n_pages, heads, page, dim, dtype, gen, device="cuda"):
    shape = (n_pages, 2, heads, page, dim)
    if dtype == ct.CT_KV_BF16:
        return torch.randn(shape, generator=gen, device=device).bfloat16(), None
    scales = (torch.rand(shape[:4], generator=gen, device=device) + 0.5) * (3.0 / QMAX[dtype])
    if dtype == ct.CT_KV_INT8:
        return torch.randint(-127, 128, shape, generator=gen, device=device, dtype=torch.int8), scales
    x = torch.randn(shape, generator=gen, device=device).mul_(120.0).clamp_(-448.0, 448.0)
    return x.to(torch.float8_e4m3fn).view(torch.uint8), scales


def make_table(lens, page, gen, window=0, spare=1, holes=()):
    """A permuted block table (device), its page count; `holes`: (sequence, logical page) left unmapped."""
    pages = [-(-int(n) // page) for n in lens]
    first = [max(0, int(n) - window) // page if window else 0 for n in lens]
    mp = max(1, max(pages) if pages else 1)
    total = sum(b - a for a, b in zip(first, pages)) + spare
    perm = torch.randperm(total, generator=gen, device="cuda").cpu().numpy()
    bt = np.full((len(lens), mp), -1, np.int32)
    at = 0
    for s in range(len(lens)):
        for lp in range(first[s], pages[s]):
            if (s, lp) not in holes:
                bt[s, lp] = perm[at]
            at += 1
    return torch.from_numpy(bt).cuda(), total


def bounds_of(k: np.ndarray):
    """Bounds codes [2][dim] and scale of a page's keys k [tokens][dim] (fp32)."""
    dim = k.shape[-1]
    if k.shape[0] == 0:
        return np.zeros((2, dim), np.int8), np.float32(0)
    if not np.isfinite(k).all():
        return np.zeros((2, dim), np.int8), np.float32(np.nan)
    hi, lo = k.max(0).astype(np.float32), k.min(0).astype(np.float32)
    s = np.float32(max(np.abs(hi).max(), np.abs(lo).max()) / np.float32(127))
    if s == 0:
        return np.zeros((2, dim), np.int8), s
    codes = np.stack((np.clip(np.ceil(hi / s), -127, 127), np.clip(np.floor(lo / s), -127, 127)))
    return codes.astype(np.int8), s


def select(q, bounds, bscales, table, lens, n_pages, page, hq, order, n_select, n_first, n_last, window=0):
    """The chosen pages by the definition, in whole numbers and single 32-bit roundings (numpy inputs)."""
    S, MP = table.shape
    H = bounds.shape[1]
    out = np.full((S, H, n_select), -1, np.int32)
    for s in range(S):
        n = min(max(int(lens[s]), 0), MP * page)
        if n == 0:
            continue
        start = max(0, n - window) if window else 0
        first, last = start // page, (n - 1) // page
        cand = [lp for lp in range(first, last + 1) if 0 <= table[s, lp] < n_pages]
        for kv in range(H):
            heads = [h for h in range(hq) if kv_head(h, hq, H, order) == kv]
            x = q[s, heads].astype(np.float32)
            with np.errstate(all="ignore"):
                e = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32)
                bad = not np.isfinite(x).all()
                c = np.where((e > 0)[:, None] & np.isfinite(e)[:, None], np.rint(x / e[:, None]), 0)
                c = np.clip(np.nan_to_num(c), -127, 127).astype(np.int64)
                b = bounds[table[s, cand], kv].astype(np.int64)
                dot = np.maximum(c, 0) @ b[:, 0].T + np.minimum(c, 0) @ b[:, 1].T
                score = ((dot.astype(np.float32) * e[:, None]).max(0) * bscales[table[s, cand], kv]).astype(np.float32)
            score = np.where(np.isnan(score) | bad, np.float32(np.inf), score)
            rank = sorted(range(len(cand)),
                          key=lambda i: (0 if cand[i] < first + n_first or cand[i] > last - n_last else 1,
                                         0.0 if cand[i] < first + n_first or cand[i] > last - n_last else -float(score[i]), i))
            got = sorted(cand[i] for i in rank[:n_select])
            out[s, kv, :len(got)] = got
    return out
