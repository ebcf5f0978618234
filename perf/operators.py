"""What the grouped-query cache operators are measured on.

The operators: writing new K and V rows into a paged cache with one scale per token and head (and reading them back),
decode attention of one new token per sequence over that cache, the page bounds and the selection of pages by a cheap
score, and decode attention over the selected pages only.

`run` computes them in plain torch operations, or with `own` through the package's entry points.  Layouts:
pool [page][K, V][kv head][slot][dim], scales [page][K, V][kv head][slot], bounds [page][kv head][upper, lower][dim],
bound scales [page][kv head], block table [sequence][logical page], q and out [sequence][query head][dim].
"""
import random

import numpy as np
import torch

own = False

DTYPES = ("bf16", "int8", "e4m3")
QMAX = {"int8": 127.0, "e4m3": 448.0}
FLT_MAX = float(np.finfo(np.float32).max)


# ---- cases ----------------------------------------------------------------------------------------------------------

def listed():
    base = dict(kv_heads=8, dim=128, page=64, dtype="bf16")
    att = dict(base, q_heads=32, window=0, order="modulo", fused=False)
    return [
        # one decode step of a server: a token of each of 64 sequences, out of a fused projection, bounds kept
        dict(base, name="write_step", op="write", tokens=64, src="bf16", fused=True, bounds=True, back=""),
        # a prompt chunk of several sequences into an int8 cache, read back as a prefix that is used again
        dict(base, name="write_prompt_int8", op="write", tokens=16384, dtype="int8", src="bf16", fused=False,
             bounds=True, back="bf16"),
        # an odd number of tokens from a model that keeps fp32, small pages, an odd number of heads
        dict(name="write_odd_e4m3", op="write", tokens=9001, kv_heads=5, dim=96, page=16, dtype="e4m3", src="f32",
             fused=False, bounds=False, back="f32"),
        # one user, a short conversation: latency
        dict(att, name="decode_one", op="decode", seqs=1, longest=777, lens="same"),
        # the ordinary serving batch, 32 sequences of 4096 tokens
        dict(att, name="decode_batch", op="decode", seqs=32, longest=4096, lens="same"),
        # a large ragged batch over an int8 cache
        dict(att, name="decode_ragged_int8", op="decode", seqs=64, longest=16384, lens="linear", dtype="int8"),
        # many short and a few longer sequences, a head each for K and V, a sliding window, one row empty
        dict(name="decode_short_e4m3", op="decode", seqs=256, longest=2500, lens="log", q_heads=12, kv_heads=12, dim=64,
             page=32, dtype="e4m3", window=1024, order="blocked", fused=True),
        # choosing 16 of 128 pages for two users
        dict(base, name="select_small", op="select", seqs=2, longest=8192, lens="same", q_heads=32, order="modulo",
             window=0, pick=16),
        # choosing 64 of up to 1024 pages for a batch of long documents
        dict(base, name="select_long", op="select", seqs=64, longest=65536, lens="linear", q_heads=32, order="modulo",
             window=0, pick=64),
        # one user with a long document, 48 pages a head: latency
        dict(att, name="selected_one", op="selected", seqs=1, longest=32768, lens="same", pick=48),
        # a batch of long documents, 64 pages a head
        dict(att, name="selected_batch", op="selected", seqs=32, longest=32768, lens="linear", pick=64),
        # wide heads in large groups over an e4m3 cache with large pages, ragged
        dict(name="selected_wide_e4m3", op="selected", seqs=24, longest=20001, lens="linear", q_heads=64, kv_heads=4,
             dim=256, page=128, dtype="e4m3", window=0, order="blocked", fused=False, pick=24),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    while True:
        op = rng.choice(("write", "decode", "decode", "select", "selected"))
        c = dict(op=op, kv_heads=rng.choice((1, 2, 3, 4, 5, 8, 12, 16)), dim=rng.choice((32, 64, 64, 96, 128, 128, 128, 192, 256)),
                 page=rng.choice((16, 32, 48, 64, 64, 128)), dtype=rng.choice(DTYPES))
        if op == "write":
            c.update(tokens=_log(rng, 1, 20000), src=rng.choice(("bf16", "f32")), fused=rng.random() < 0.5,
                     bounds=rng.random() < 0.5)
            c["back"] = rng.choice(("bf16", "f32")) if c["dtype"] != "bf16" or rng.random() < 0.5 else ""
        else:
            c.update(seqs=_log(rng, 1, 256), longest=_log(rng, 1, 65536), lens=rng.choice(("same", "linear", "log")),
                     q_heads=c["kv_heads"] * rng.choice((1, 2, 3, 4, 7, 8, 16)), order=rng.choice(("modulo", "blocked")),
                     window=rng.choice((0, 0, 0, _log(rng, 1, 8192))))
            if op == "select":
                c["dtype"] = "bf16"
            else:
                c["fused"] = rng.random() < 0.5
            if op != "decode":
                c["pick"] = _log(rng, 4, 128)
            if op == "select":                        # there is something to choose
                reach = min(c["longest"], c["window"] or c["longest"])
                if reach < 2 * c["pick"] * c["page"] or c["seqs"] * c["kv_heads"] * c["pick"] < 24:
                    continue
        w = work(c)
        # no dearer than the largest listed case, and its plain form (which pads to the longest) fits the card
        padded = 0 if op == "write" else c["seqs"] * (min(c["longest"] + c["page"], c["pick"] * c["page"])
                                                      if op == "selected" else c["longest"] + c["page"]) * c["kv_heads"] * c["dim"]
        held = 0 if op in ("write", "select") else sum(_lens(c)) * c["kv_heads"] * c["dim"]
        if w["bytes"] <= 1.0e9 and max(padded if op != "select" else padded // c["page"] * 16, held // 4) <= 1.1e9:
            return c


def _lens(c):
    n, top = c["seqs"], c["longest"]
    if c["lens"] == "same":
        return [top] * n
    if c["lens"] == "linear":
        return [max(1, top * (i + 1) // n) for i in range(n)]
    lens = [max(1, int(round(top ** ((i + 1) / n)))) for i in range(n)]
    if n >= 8:
        lens[0] = 0                                   # a row of the batch that no sequence uses now
    return lens


def _elt(dtype):
    return 2 if dtype == "bf16" else 1


def work(c):
    H, D, P = c["kv_heads"], c["dim"], c["page"]
    row = D * _elt(c["dtype"]) + (0 if c["dtype"] == "bf16" else 4)          # one stored K or V row
    if c["op"] == "write":
        n, src = c["tokens"], 2 if c["src"] == "bf16" else 4
        b = n * H * 2 * (D * src + row) + 4 * n
        if c["back"]:
            b += n * H * 2 * (row + D * (2 if c["back"] == "bf16" else 4)) + 4 * n
        if c["bounds"]:
            m = _touched(c)
            b += m * H * (2 * D + 4) + 8 * m          # the keys are in hand when their bounds are made
        return {"bytes": b, "flops": 4 * n * H * D}
    Hq = c["q_heads"]
    tokens = pages = 0
    for n in _lens(c):
        first = max(0, n - c["window"]) if c["window"] else 0
        have = -(-n // P) - first // P if n else 0
        if c["op"] == "selected" and have > c["pick"]:
            tokens += min(c["pick"] * P, n - first)
            pages += c["pick"]
        else:
            tokens += n - first
            pages += have
    S = c["seqs"]
    q = S * Hq * D * 2
    if c["op"] == "select":
        return {"bytes": pages * (H * (2 * D + 4) + 4) + q + S * H * c["pick"] * 4 + 4 * S, "flops": 4 * pages * Hq * D}
    b = tokens * H * 2 * row + 2 * q + S * Hq * 4 + 4 * S + 4 * pages * (H if c["op"] == "selected" else 1)
    return {"bytes": b, "flops": 4 * tokens * Hq * D}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _touched(c):
    """Pages that a write of c["tokens"] tokens to runs of a page's slots reaches."""
    return -(-c["tokens"] // c["page"]) if c["tokens"] > c["page"] else c["tokens"]


def _pool(c, n_pages, gen):
    shape = (n_pages, 2, c["kv_heads"], c["page"], c["dim"])
    dev = "cuda"
    if c["dtype"] == "bf16":
        return torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16), None
    scales = (torch.rand(shape[:4], generator=gen, device=dev) + 0.5) * (3.0 / QMAX[c["dtype"]])
    if c["dtype"] == "int8":
        return torch.randint(-127, 128, shape, generator=gen, device=dev, dtype=torch.int8), scales
    x = torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16).mul_(120.0).clamp_(-448.0, 448.0)
    return x.to(torch.float8_e4m3fn).view(torch.uint8), scales


def _rows(n, heads, dim, n_other, dtype, fused, gen):
    """[n][heads * dim] values; fused: the first columns of a wider matrix, as a projection of q, k and v gives them."""
    wide = torch.randn(n, heads * dim + (n_other if fused else 0), generator=gen, device="cuda", dtype=torch.float32)
    return wide.to(torch.bfloat16 if dtype == "bf16" else torch.float32)


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    H, D, P = c["kv_heads"], c["dim"], c["page"]
    s = {"c": c, "gen_seed": int(seed)}
    if c["op"] == "write":
        n, m = c["tokens"], _touched(c)
        n_pages = m + 3
        s["pool"], s["scales"] = _pool(c, n_pages, gen)
        pages = torch.randperm(n_pages, generator=gen, device="cuda")[:m]
        if n > P:                                     # whole pages, the last one in part
            t = torch.arange(n, device="cuda")
            page, slot = pages[t // P], t % P
            counts = torch.full((m,), P, device="cuda")
            counts[-1] = n - (m - 1) * P
        else:                                         # the newest token of one page each
            page, slot = pages, torch.randint(0, P, (n,), generator=gen, device="cuda")
            counts = slot + 1
        s["slots"] = (page * P + slot).to(torch.int32)
        s["pages"], s["counts"] = pages.to(torch.int32), counts.to(torch.int32)
        both = _rows(n, 2 * H, D, 4 * H * D, c["src"], c["fused"], gen)
        # keys with channels of their own size and offset, and a few large tokens
        size = torch.rand(H * D, generator=gen, device="cuda") * 2 + 0.25
        both[:, :H * D] = both[:, :H * D] * size + torch.randn(H * D, generator=gen, device="cuda")
        both[torch.rand(n, generator=gen, device="cuda") < 0.01] *= 20.0
        s["k"], s["v"] = both[:, :H * D], both[:, H * D:2 * H * D]
        s["bounds"] = torch.zeros(n_pages, H, 2, D, device="cuda", dtype=torch.int8)
        s["bound_scales"] = torch.zeros(n_pages, H, device="cuda")
        if c["back"]:
            t = torch.bfloat16 if c["back"] == "bf16" else torch.float32
            s["k_back"] = torch.empty(n, H * D, device="cuda", dtype=t)
            s["v_back"] = torch.empty(n, H * D, device="cuda", dtype=t)
        if own:
            s["layout"] = _layout(c, n_pages, 1)
        return s
    S, Hq = c["seqs"], c["q_heads"]
    order = random.Random(int(seed))
    lens = _lens(c)
    order.shuffle(lens)
    pages = [-(-n // P) for n in lens]
    first = [max(0, n - c["window"]) // P if c["window"] else 0 for n in lens]
    live = [b - a for a, b in zip(first, pages)]      # pages wholly before the window are gone, as the cache frees them
    MP = max(1, max(pages))
    n_pages = sum(live) + 2
    perm = torch.randperm(n_pages, generator=gen, device="cuda").cpu().numpy().astype(np.int32)
    bt = np.full((S, MP), -1, np.int32)
    at = 0
    for i in range(S):
        bt[i, first[i]:pages[i]] = perm[at:at + live[i]]
        at += live[i]
    s["table"] = torch.from_numpy(bt).cuda()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = _rows(S, Hq, D, 2 * H * D, "bf16", c.get("fused", False), gen)
    s["q"] = q[:, :Hq * D]
    if c["op"] == "select":
        # bounds of pages whose keys drift from page to page, rounded outward
        mid = torch.randn(n_pages, H, D, generator=gen, device="cuda")
        half = torch.rand(n_pages, H, D, generator=gen, device="cuda") * 2 + 0.5
        scale = (mid.abs() + half).amax(-1) / 127
        s["bounds"] = torch.stack((torch.ceil((mid + half) / scale[..., None]), torch.floor((mid - half) / scale[..., None])),
                                  2).clamp_(-127, 127).to(torch.int8)
        s["bound_scales"] = scale
        s["picked"] = torch.empty(S, H, c["pick"], device="cuda", dtype=torch.int32)
    else:
        s["pool"], s["scales"] = _pool(c, n_pages, gen)
        for i, n in enumerate(lens):                  # what lies behind a sequence's end is not its own
            if n % P and i % 7 == 0:
                tail = int(bt[i, pages[i] - 1])
                (s["pool"] if c["dtype"] == "bf16" else s["scales"])[tail, :, :, n % P:] = float("nan")
        if c["op"] == "selected":
            pick = c["pick"]
            key = torch.rand(S, H, MP, generator=gen, device="cuda")
            lp = torch.arange(MP, device="cuda")
            inside = (lp[None] >= torch.tensor(first, device="cuda")[:, None]) & (lp[None] < torch.tensor(pages, device="cuda")[:, None])
            key = torch.where(inside[:, None], key, torch.full_like(key, 2.0))
            got = key.argsort(-1)[..., :pick]
            got = torch.where(key.gather(-1, got) < 1.5, got, torch.full_like(got, MP)).sort(-1).values
            got = torch.where(got < MP, got, torch.full_like(got, -1))
            if got.shape[-1] < pick:
                got = torch.cat((got, torch.full((S, H, pick - got.shape[-1]), -1, device="cuda")), -1)
            s["picked"] = got.to(torch.int32).contiguous()
        s["out"] = torch.empty(S, Hq, D, device="cuda", dtype=torch.bfloat16)
        s["lse"] = torch.empty(S, Hq, device="cuda")
    if own:
        s["plan"] = _plan(c, S, n_pages, MP)
    return s


# ---- the package's calls ----------------------------------------------------------------------------------------------

def _layout(c, n_pages, max_pages):
    import cautreo_b200 as ct
    kind = {"bf16": ct.CT_KV_BF16, "int8": ct.CT_KV_INT8, "e4m3": ct.CT_KV_E4M3}[c["dtype"]]
    return ct.GqaLayout(c["kv_heads"], c["dim"], c["page"], kind, n_pages, max_pages)


def _plan(c, n_seq, n_pages, max_pages):
    import cautreo_b200 as ct
    order = ct.CT_GQA_MODULO if c["order"] == "modulo" else ct.CT_GQA_BLOCKED
    return ct.GqaPlan(_layout(c, n_pages, max_pages), n_seq, c["q_heads"], window_tokens=c["window"], head_order=order)


def _run_own(s):
    import cautreo_b200 as ct
    c = s["c"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "write":
        kind = {"bf16": ct.CT_KV_BF16, "f32": ct.CT_KV_F32}
        n = c["tokens"]
        ct.gqa_write_slots(s["layout"], s["pool"], s["scales"], s["k"], s["v"], s["slots"], n, src_dtype=kind[c["src"]],
                           k_stride=s["k"].stride(0), v_stride=s["v"].stride(0), stream=stream)
        if c["bounds"]:
            ct.gqa_page_bounds(s["layout"], s["pool"], s["scales"], s["pages"], s["counts"], s["pages"].numel(), s["bounds"],
                               s["bound_scales"], stream=stream)
        if c["back"]:
            ct.gqa_read_slots(s["layout"], s["pool"], s["scales"], s["slots"], n, s["k_back"], s["v_back"],
                              out_dtype=kind[c["back"]], stream=stream)
        return _write_outputs(s)
    if c["op"] == "select":
        s["plan"].select(s["q"], s["bounds"], s["bound_scales"], s["table"], s["lens"], s["picked"], c["pick"], n_first=1,
                         n_last=1, q_stride=s["q"].stride(0), stream=stream)
        return s["picked"]
    if c["op"] == "selected":
        s["plan"].decode_selected(s["q"], s["pool"], s["scales"], s["table"], s["lens"], s["picked"], c["pick"], s["out"],
                                  s["lse"], q_stride=s["q"].stride(0), stream=stream)
    else:
        s["plan"].decode(s["q"], s["pool"], s["scales"], s["table"], s["lens"], s["out"], s["lse"],
                         q_stride=s["q"].stride(0), stream=stream)
    return s["out"], s["lse"]


def _write_outputs(s):
    out = {"k": s["k_back"], "v": s["v_back"]} if s["c"]["back"] else {"pool": s["pool"]}
    if s["c"]["bounds"]:
        out["bounds"], out["bound_scales"] = s["bounds"], s["bound_scales"]
    return out


# ---- the plain forms ----------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _run_own(s)
    op = s["c"]["op"]
    return _plain_write(s) if op == "write" else _plain_select(s) if op == "select" else _plain_attention(s)


def _encode(x, dtype):
    """Codes and scales of rows x [..., dim] in fp32: one scale a row; a row with a NaN or an infinity has scale NaN."""
    if dtype == "bf16":
        return x.to(torch.bfloat16), None
    top = x.abs().amax(-1, keepdim=True)
    d = top / torch.full_like(top, QMAX[dtype])
    inv = torch.where(d > 0, (1.0 / d).clamp(max=FLT_MAX), torch.zeros_like(d))
    fine = torch.isfinite(top)
    y = torch.where(fine, x, torch.zeros_like(x)) * inv
    if dtype == "int8":
        codes = torch.floor(y + 0.5).clamp(-127, 127).to(torch.int8)
    else:
        codes = y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(fine, codes, torch.zeros_like(codes))
    return codes, torch.where(fine, d, torch.full_like(d, float("nan")))[..., 0]


def _values(codes, scales, dtype):
    if dtype == "bf16":
        return codes.float()
    x = codes.float() if dtype == "int8" else codes.view(torch.float8_e4m3fn).float()
    return x * scales[..., None]


def _plain_write(s):
    c = s["c"]
    H, D, P, n = c["kv_heads"], c["dim"], c["page"], c["tokens"]
    pool, scales, dt = s["pool"], s["scales"], c["dtype"]
    page, slot = s["slots"].long() // P, s["slots"].long() % P
    rows = torch.stack((s["k"], s["v"]), 1).float().view(n, 2, H, D)
    codes, sc = _encode(rows, dt)
    pool.permute(0, 3, 1, 2, 4)[page, slot] = codes
    if sc is not None:
        scales.permute(0, 3, 1, 2)[page, slot] = sc
    if c["bounds"]:
        pages = s["pages"].long()
        k = _values(pool[pages, 0], None if scales is None else scales[pages, 0], dt)            # [m][H][P][D]
        live = torch.arange(P, device="cuda")[None] < s["counts"][:, None]
        live = live[:, None, :, None]
        hi = torch.where(live, k, torch.full_like(k, float("-inf"))).amax(2)
        lo = torch.where(live, k, torch.full_like(k, float("inf"))).amin(2)
        top = torch.maximum(hi.abs(), lo.abs()).amax(-1, keepdim=True)
        d = top / torch.full_like(top, 127.0)
        up = torch.where(d > 0, torch.ceil(hi / d).clamp(-127, 127), torch.zeros_like(hi))
        down = torch.where(d > 0, torch.floor(lo / d).clamp(-127, 127), torch.zeros_like(lo))
        s["bounds"][pages] = torch.stack((up, down), 2).to(torch.int8)
        s["bound_scales"][pages] = d[..., 0]
    if c["back"]:
        got = _values(pool.permute(0, 3, 1, 2, 4)[page, slot],
                      None if scales is None else scales.permute(0, 3, 1, 2)[page, slot], dt)
        s["k_back"].copy_(got[:, 0].reshape(n, H * D))
        s["v_back"].copy_(got[:, 1].reshape(n, H * D))
    return _write_outputs(s)


def _grouped(q, c):
    """[seq][kv head][head of its group][dim] in fp32."""
    S, H, D = q.shape[0], c["kv_heads"], c["dim"]
    G = c["q_heads"] // H
    if c["order"] == "modulo":
        return q.float().reshape(S, G, H, D).transpose(1, 2)
    return q.float().reshape(S, H, G, D)


def _ungrouped(x, c):
    """[seq][kv head][head of its group][...] -> [seq][query head][...]."""
    if c["order"] == "modulo":
        x = x.transpose(1, 2)
    return x.reshape(x.shape[0], c["q_heads"], *x.shape[3:])


def _plain_select(s):
    c = s["c"]
    n, window, pick = s["lens"].long(), c["window"], c["pick"]
    table = s["table"].long()
    S, MP = table.shape
    q = _grouped(s["q"], c)
    top = q.abs().amax(-1, keepdim=True)
    e = top / torch.full_like(top, 127.0)
    code = torch.where(e > 0, torch.round(q / e).clamp(-127, 127), torch.zeros_like(q)).double()
    code = torch.cat((code.clamp(min=0), code.clamp(max=0)), -1)                                 # [S][H][G][2 D]
    b = s["bounds"][table.clamp(min=0)].double().flatten(3).transpose(1, 2)                      # [S][H][MP][2 D]
    dot = torch.matmul(code, b.transpose(2, 3))                                                  # whole numbers: exact
    score = (dot.float() * e).amax(2) * s["bound_scales"][table.clamp(min=0)].transpose(1, 2)    # [S][H][MP]
    score = torch.where(torch.isnan(score), torch.full_like(score, float("inf")), score).double().clamp(-1e300, 1e300)
    lp = torch.arange(MP, device="cuda")[None]
    last = (n - 1).div(c["page"], rounding_mode="floor")[:, None]
    first = ((n - window).clamp(min=0) if window else torch.zeros_like(n)).div(c["page"], rounding_mode="floor")[:, None]
    inside = (lp >= first) & (lp <= last) & (table >= 0)
    kept = inside & ((lp == first) | (lp == last))
    score = torch.where(kept[:, None], torch.full_like(score, float("inf")), score)
    score = torch.where(inside[:, None], score, torch.full_like(score, float("-inf")))
    best = torch.sort(score, dim=-1, descending=True, stable=True)
    at = torch.where(best.values > float("-inf"), best.indices, torch.full_like(best.indices, MP))[..., :pick].sort(-1).values
    at = torch.where(at < MP, at, torch.full_like(at, -1)).to(torch.int32)
    s["picked"].fill_(-1)
    s["picked"][..., :at.shape[-1]] = at
    return s["picked"]


def _plain_attention(s):
    c = s["c"]
    H, D, P = c["kv_heads"], c["dim"], c["page"]
    table = s["table"].long()
    S, MP = table.shape
    lp = s["picked"].long() if c["op"] == "selected" else torch.arange(MP, device="cuda").expand(S, H, MP)
    phys = torch.where(lp >= 0, table[:, None].expand(S, H, MP).gather(2, lp.clamp(min=0)), torch.full_like(lp, -1))
    pos = lp[..., None] * P + torch.arange(P, device="cuda")                                     # [S][H][pages][P]
    n = s["lens"].long()[:, None, None, None]
    live = (phys >= 0)[..., None] & (pos < n)
    if c["window"]:
        live = live & (pos >= n - c["window"])
    live = live.reshape(S, H, 1, -1)
    at, head = phys.clamp(min=0), torch.arange(H, device="cuda")[None, :, None]

    def rows(which):
        x = _values(s["pool"][at, which, head], None if s["scales"] is None else s["scales"][at, which, head], c["dtype"])
        return x.reshape(S, H, -1, D).masked_fill_(~live.transpose(2, 3), 0.0)

    score = torch.matmul(_grouped(s["q"], c), rows(0).transpose(2, 3)) * (1.0 / float(np.sqrt(D)))
    score = score.masked_fill(~live, float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, rows(1)) / torch.where(total > 0, total, torch.ones_like(total))
    s["out"].copy_(_ungrouped(out, c))
    s["lse"].copy_(_ungrouped((top + torch.log(total))[..., 0], c))
    return s["out"], s["lse"]


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------

def _stored(codes, scales, dtype):
    x = codes.view(torch.float8_e4m3fn) if dtype == "e4m3" else codes
    return x.double() if scales is None else x.double() * scales.double().unsqueeze(-1)


def exact(case, seed):
    c = dict(case)
    if c["op"] == "select":
        return None                                   # whole numbers: compared with the plain form, where they have to be equal
    s = prepare(c, seed)
    H, D, P, dt = c["kv_heads"], c["dim"], c["page"], c["dtype"]
    if c["op"] == "write":
        if dt == "bf16" and not c["back"]:
            pool = s["pool"].double()
            for which, x in enumerate((s["k"], s["v"])):
                rounded = x.bfloat16().double().view(-1, H, D)
                pool[s["slots"].long() // P, which, :, s["slots"].long() % P] = rounded
            out = {"pool": pool}
        else:
            out = {}
            for name, x in (("k", s["k"]), ("v", s["v"])):
                x = x.double().reshape(-1, H, D)
                if dt == "bf16":
                    y = x.bfloat16().double()
                else:                                 # which code a value gets is defined by single roundings to 32 bits
                    r = x.float().cpu().numpy()
                    d = np.abs(r).max(-1, keepdims=True) / np.float32(QMAX[dt])
                    r = r * np.where(d > 0, np.float32(1) / np.maximum(d, np.float32(1e-38)), np.float32(0))
                    if dt == "int8":
                        r = np.clip(np.floor(r + np.float32(0.5)), -127, 127)
                    else:
                        r = torch.from_numpy(np.clip(r, -448, 448)).to(torch.float8_e4m3fn).double().numpy()
                    y = torch.from_numpy(r.astype(np.float64) * d.astype(np.float64)).cuda()
                out[name] = y.reshape(-1, H * D)
        if c["bounds"]:
            out["bounds"] = out["bound_scales"] = None
        return out
    lens, table = s["lens"].tolist(), s["table"]
    S, Hq = c["seqs"], c["q_heads"]
    out = torch.zeros(S, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((S, Hq), float("-inf"), dtype=torch.float64, device="cuda")
    if sum(lens) * H > 4_000_000 and c["op"] == "selected" and S * H > 4096:
        return None
    hmap = [[h for h in range(Hq) if (h % H if c["order"] == "modulo" else h * H // Hq) == kv] for kv in range(H)]
    hmap = torch.tensor(hmap, device="cuda")                                                     # [H][G]
    for i, n in enumerate(lens):
        if n == 0:
            continue
        start = max(0, n - c["window"]) if c["window"] else 0
        if c["op"] == "selected":
            pages = s["picked"][i].long()                                                        # [H][pick]
        else:
            pages = torch.arange(start // P, -(-n // P), device="cuda").expand(H, -1)
        pos = (pages.unsqueeze(-1) * P + torch.arange(P, device="cuda")).flatten(1)              # [H][T]
        ok = (pages >= 0).unsqueeze(-1).expand(-1, -1, P).flatten(1) & (pos < n) & (pos >= start)
        phys = table[i].long()[pages.clamp_min(0)]
        heads = torch.arange(H, device="cuda").unsqueeze(1)
        kv = []
        for which in (0, 1):
            sc = None if s["scales"] is None else s["scales"][phys, which, heads]
            kv.append(torch.where(ok.unsqueeze(-1), _stored(s["pool"][phys, which, heads], sc, dt).flatten(1, 2), 0.0))
        qi = s["q"][i].double().view(Hq, D)[hmap]                                                # [H][G][D]
        logit = torch.einsum("hgd,htd->hgt", qi, kv[0]) / D ** 0.5
        logit = torch.where(ok.unsqueeze(1), logit, float("-inf"))
        weight = torch.softmax(logit, -1)
        out[i, hmap] = torch.einsum("hgt,htd->hgd", weight, kv[1])
        lse[i, hmap] = torch.logsumexp(logit, -1)
    return out, lse
