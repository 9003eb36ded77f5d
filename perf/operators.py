"""The serving operators as measured: the sliding-window prompt attention, the
8-bit paged K/V cache's append, its single-token attention and its page copy.

``run`` is one pass: the plain torch form of the operator, or, with ``own``
set, the framework's call through ``vkcuda_b200.vc``. Shapes follow the
attention workloads of the benchmark (16 and 32 heads, 4096 and 8192 tokens,
head dims 64 and 128) and their serving counterparts.
"""
import math

import torch

own = False

LOG2E = 1.4426950408889634
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
E4M3_MAX = 448.0
NAN_CODE = 0x7F


def listed():
    return [
        # A short prompt of a small model: launch latency counts.
        dict(name="window_short", op="window", B=1, Hq=8, Hkv=2, Nq=97, Nk=97, d=64, window=64,
             sinks=4, dtype="fp16", tokens_first=False, ragged=False),
        # A padded batch of prompts as the projection leaves it (token-major), 1K window.
        dict(name="window_batch", op="window", B=4, Hq=16, Hkv=4, Nq=4000, Nk=4000, d=128,
             window=1024, sinks=4, dtype="fp16", tokens_first=True, ragged=True),
        # The second chunk of a long prompt against everything before it, wide window.
        dict(name="window_chunk", op="window", B=2, Hq=32, Hkv=8, Nq=2048, Nk=6144, d=128,
             window=4096, sinks=16, dtype="bf16", tokens_first=True, ragged=False),
        # One long prompt, whole.
        dict(name="window_long", op="window", B=1, Hq=32, Hkv=8, Nq=8192, Nk=8192, d=128,
             window=2048, sinks=4, dtype="bf16", tokens_first=False, ragged=False),
        # A decode step: one new token for each of 32 sequences.
        dict(name="append_step", op="append", B=32, new=1, start=4096, Hkv=8, d=128, page=64,
             dtype="bf16", ragged=False),
        # Ragged prompts appended behind a shared, partly filled prefix.
        dict(name="append_prompts", op="append", B=8, new=8193, start=100, Hkv=8, d=128, page=32,
             dtype="fp16", ragged=True),
        # One sequence, a few heads, a short context: latency.
        dict(name="attn_short", op="attn", B=1, Hq=8, Hkv=2, d=64, page=16, length=500, window=0,
             sinks=0, dtype="fp16", ragged=False),
        # An ordinary decode batch of uneven sequences.
        dict(name="attn_batch", op="attn", B=32, Hq=32, Hkv=8, d=128, page=64, length=16384,
             window=0, sinks=0, dtype="bf16", ragged=True),
        # Long sequences read through a window with sinks.
        dict(name="attn_window", op="attn", B=64, Hq=16, Hkv=4, d=128, page=32, length=16384,
             window=4096, sinks=4, dtype="fp16", ragged=True),
        # Few very long sequences: the work has to be split along the tokens.
        dict(name="attn_long", op="attn", B=2, Hq=16, Hkv=1, d=128, page=128, length=131072,
             window=0, sinks=0, dtype="bf16", ragged=True),
        # A fork: the last, partly filled page of a few sequences, every layer.
        dict(name="copy_fork", op="copy", layers=16, Hkv=8, d=128, page=64, pages=64, n=8),
        # A compaction that moves many pages.
        dict(name="copy_compact", op="copy", layers=8, Hkv=8, d=128, page=32, pages=2048, n=900),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "append", "attn", "copy"])
    d, dtype = rng.choice([64, 128]), rng.choice(["fp16", "bf16"])
    Hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 7, 8, 16])
    if op == "window":
        Hq = min(Hkv * group, 32) // Hkv * Hkv
        Nk = _log(rng, 16, 8192)
        Nq = Nk if rng.random() < 0.6 else _log(rng, 1, Nk)
        B = max(1, min(_log(rng, 1, 8), 32 * 8192 * 8192 // (2 * Hq * Nq * Nk)))
        case = dict(op=op, B=B, Hq=Hq, Hkv=Hkv, Nq=Nq, Nk=Nk, d=d,
                    window=rng.choice([0, _log(rng, 1, 4096), _log(rng, 64, 4096)]),
                    sinks=rng.choice([0, 1, 4, 130]), dtype=dtype,
                    tokens_first=rng.random() < 0.5, ragged=rng.random() < 0.4)
        most = max(work(c)["flops"] for c in listed() if c["op"] == op)
        while work(case)["flops"] > most:
            case["Nq"] = case["Nq"] * 3 // 4
        return case
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        if rng.random() < 0.4:
            return dict(op=op, B=_log(rng, 1, 256), new=1, start=_log(rng, 1, 2000), Hkv=Hkv, d=d,
                        page=page, dtype=dtype, ragged=False)
        B = _log(rng, 1, 16)
        return dict(op=op, B=B, new=_log(rng, 2, 32768 // B), start=rng.choice([0, 17, 1000]),
                    Hkv=Hkv, d=d, page=page, dtype=dtype, ragged=rng.random() < 0.5)
    if op == "attn":
        B = _log(rng, 1, 64)
        return dict(op=op, B=B, Hq=Hkv * group, Hkv=Hkv, d=d, page=page,
                    length=_log(rng, 1, min(131072, 262144 // max(B, Hkv))),
                    window=rng.choice([0, 0, _log(rng, 1, 8192)]), sinks=rng.choice([0, 4, 100]),
                    dtype=dtype, ragged=rng.random() < 0.7)
    pages = _log(rng, 16, 2048)
    return dict(op=op, layers=rng.choice([1, 2, 4, 8]), Hkv=Hkv, d=d, page=min(page, 32),
                pages=pages, n=max(1, int(pages * rng.uniform(0.02, 0.45))))


# ------------------------------------------------------------------ lengths
def _spread(case, most, key="ragged"):
    """The sequences' lengths: all `most`, or spread over [most / 8, most]."""
    if not case[key]:
        return [most] * case["B"]
    return [max(1, int(most * (0.125 + 0.875 * ((0.37 + 0.6180339887 * b) % 1.0))))
            for b in range(case["B"])]


def _visible(pos, window, sinks):
    """Keys that the token at position `pos` sees."""
    if pos < 0:
        return 0
    if window == 0 or pos + 1 <= window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def _pairs(Nq, Nk, length, window, sinks):
    return sum(_visible(p, window, sinks) for p in range(Nk - Nq, min(Nk, length)))


def work(case):
    if case["op"] == "window":
        lens = _spread(case, case["Nk"])
        pairs = sum(_pairs(case["Nq"], case["Nk"], n, case["window"], case["sinks"]) for n in lens)
        rows = case["B"] * case["d"] * 2
        return {"bytes": rows * (2 * case["Hq"] * case["Nq"] + 2 * case["Hkv"] * case["Nk"]),
                "flops": 4 * case["d"] * case["Hq"] * pairs}
    if case["op"] == "append":
        tokens = sum(_spread(case, case["new"]))
        return {"bytes": tokens * case["Hkv"] * case["d"] * 2 * (2 + 1), "flops": 0}
    if case["op"] == "attn":
        lens = _spread(case, case["length"])
        seen = sum(_visible(n - 1, case["window"], case["sinks"]) for n in lens)
        return {"bytes": seen * case["Hkv"] * case["d"] * 2 + case["B"] * case["Hq"] * case["d"] * 4,
                "flops": 4 * case["d"] * case["Hq"] * seen}
    one = case["Hkv"] * case["page"] * case["d"] * 2 + case["Hkv"] * 8
    return {"bytes": 2 * case["layers"] * case["n"] * one, "flops": 0}


# ------------------------------------------------------------------ states
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _shuffled(values, g, dtype=torch.int32):
    order = torch.randperm(len(values), device="cuda", generator=g)
    return torch.tensor(values, dtype=dtype, device="cuda")[order].contiguous()


def _table(lens, page, spare, g):
    """A page table of scattered pages: row b holds the pages of lens[b] tokens, -1 behind them."""
    B = lens.numel()
    need = (lens.long() + page - 1) // page
    width = max(1, int(need.max()))
    total = int(need.sum()) + spare
    ids = torch.randperm(total, device="cuda", generator=g).to(torch.int32)
    col = torch.arange(width, device="cuda")
    held = col[None, :] < need[:, None]
    first = torch.cumsum(need, 0) - need
    slot = (first[:, None] + col[None, :]).clamp_(max=max(total - 1, 0))
    return torch.where(held, ids[slot], torch.full_like(slot, -1, dtype=torch.int32)).contiguous(), total


def _cache(total, case, g):
    """Codes and scales as an append leaves them: values of unit size in e4m3, one scale per page
    and head (K, V apart)."""
    H, P, d = case["Hkv"], case["page"], case["d"]
    state = {}
    for x in "kv":
        codes = torch.empty(total, H, P, d, dtype=torch.float8_e4m3fn, device="cuda")
        step = max(1, (1 << 27) // (H * P * d))
        for i in range(0, total, step):
            n = min(step, total - i)
            codes[i:i + n] = (_randn(g, n, H, P, d) * 110).clamp_(-448, 448).to(torch.float8_e4m3fn)
        state[x] = codes
        state[x + "s"] = torch.rand(total, H, device="cuda", generator=g) * 0.01 + 0.004
    return state


def _nan_tails(codes, table, lens, page):
    """NaN codes in the slots behind each sequence's last token: an old page's leavings."""
    last = ((lens.long() - 1) // page).clamp_(min=0)
    ids = table.gather(1, last[:, None])[:, 0].long()
    slot = torch.arange(page, device="cuda")
    bad = slot[None, :] > ((lens.long() - 1) % page)[:, None]
    raw = codes.view(torch.uint8)
    rows = raw[ids]
    rows = torch.where(bad[:, None, :, None], torch.full_like(rows, NAN_CODE), rows)
    raw[ids] = rows


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case, "op": case["op"]}
    if case["op"] == "window":
        B, Hq, Hkv, Nq, Nk, d = (case[k] for k in ("B", "Hq", "Hkv", "Nq", "Nk", "d"))
        t = TYPES[case["dtype"]]

        def make(H, N):
            x = _randn(g, B, N, H, d) if case["tokens_first"] else _randn(g, B, H, N, d)
            x = x.to(t)
            return x.transpose(1, 2) if case["tokens_first"] else x

        s["q"], s["k"], s["v"] = make(Hq, Nq), make(Hkv, Nk), make(Hkv, Nk)
        s["o"] = torch.zeros_like(s["q"])
        s["lens"] = _shuffled(_spread(case, Nk), g) if case["ragged"] else None
        if s["lens"] is not None:  # the padding holds what an earlier batch left
            pad = torch.arange(Nk, device="cuda")[None, :] >= s["lens"][:, None]
            for x in ("k", "v"):
                s[x].masked_fill_(pad[:, None, :, None], float("nan"))
        s["scale"] = LOG2E / math.sqrt(d)
        if own:
            s["strides"] = [s[x].stride()[:3] for x in ("q", "k", "v", "o")]
        return s
    if case["op"] == "append":
        t = TYPES[case["dtype"]]
        low = case["start"] // 2
        both = [n << 32 | (low + 7919 * b % (case["start"] + 1 - low))
                for b, n in enumerate(_spread(case, case["new"]))]
        both = _shuffled(both, g, torch.int64)
        new, s["start"] = (both >> 32).to(torch.int32), (both & 0xFFFFFFFF).to(torch.int32)
        s["table"], total = _table(s["start"] + new, case["page"], 3, g)
        s.update(_cache(total, case, g))
        for x in "kv":  # an append leaves scales that are powers of two
            s[x + "s"] = torch.exp2(torch.floor(torch.log2(s[x + "s"])))
        s["cu"] = torch.cat([new.new_zeros(1), torch.cumsum(new, 0, dtype=torch.int32)])
        s["tokens"] = int(new.sum())
        s["most"] = int(new.max())
        # Some tokens are far larger than those before them, as the first ones of a text are.
        size = torch.exp2(torch.randint(-2, 5, (s["tokens"], 1, 1), device="cuda", generator=g).float())
        s["kn"] = (_randn(g, s["tokens"], case["Hkv"], case["d"]) * size).to(t)
        s["vn"] = _randn(g, s["tokens"], case["Hkv"], case["d"]).to(t)
        s["lens"] = torch.zeros_like(s["start"])
        if own:
            s["cache"] = _handle(s, case)
        return s
    if case["op"] == "attn":
        s["lens"] = _shuffled(_spread(case, case["length"]), g)
        s["table"], total = _table(s["lens"], case["page"], 3, g)
        s.update(_cache(total, case, g))
        for x in "kv":
            _nan_tails(s[x], s["table"], s["lens"], case["page"])
        s["q"] = _randn(g, case["B"], case["Hq"], case["d"]).to(TYPES[case["dtype"]])
        s["o"] = torch.empty_like(s["q"])
        s["scale"] = LOG2E / math.sqrt(case["d"])
        if own:
            from vkcuda_b200 import vc
            s["cache"] = _handle(s, case)
            err, need = vc.kv8_attn_workspace(s["cache"], case["B"], case["Hq"])
            vc.check(err, "kv8_attn_workspace")
            s["ws"] = torch.zeros(need, dtype=torch.uint8, device="cuda")
        return s
    L, H, P, d, pages = (case[k] for k in ("layers", "Hkv", "page", "d", "pages"))
    for x in "kv":
        s[x] = torch.randint(0, 256, (L, pages, H, P, d), device="cuda", generator=g, dtype=torch.uint8)
        s[x + "s"] = torch.rand(L, pages, H, device="cuda", generator=g)
    ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    s["src"], s["dst"] = ids[:case["n"]].contiguous(), ids[case["n"]:2 * case["n"]].contiguous()
    if own:
        from vkcuda_b200 import vc
        s["caches"] = vc.kv8_layers([vc.kv8_cache(s["k"][i], s["v"][i], s["ks"][i], s["vs"][i], pages,
                                                  H, P, d) for i in range(L)])
    return s


def _handle(s, case):
    from vkcuda_b200 import vc
    return vc.kv8_cache(s["k"], s["v"], s["ks"], s["vs"], s["k"].shape[0], case["Hkv"], case["page"],
                        case["d"])


# ------------------------------------------------------------------ passes
def run(state):
    return {"window": _window, "append": _append, "attn": _attn, "copy": _copy}[state["op"]](state)


def _weights(scores, seen):
    """Numerators and denominators of a softmax over the last axis in base 2, rows without a key: 0."""
    scores = scores.masked_fill(~seen, float("-inf"))
    most = scores.amax(-1, keepdim=True)
    p = torch.exp2(scores - torch.where(torch.isinf(most), torch.zeros_like(most), most))
    return p, p.sum(-1, keepdim=True)


def _window(s):
    c = s["case"]
    B, Hq, Hkv, Nq, Nk, d = (c[k] for k in ("B", "Hq", "Hkv", "Nq", "Nk", "d"))
    if own:
        from vkcuda_b200 import vc
        q, k, v, o = s["strides"]
        vc.check(vc.flash_window_fwd(s["q"], s["k"], s["v"], s["o"], B, Hq, Hkv, Nq, Nk, d, s["scale"],
                                     vc.Dtype.F16 if c["dtype"] == "fp16" else vc.Dtype.BF16,
                                     window=c["window"], sinks=c["sinks"], lens=s["lens"], q_strides=q,
                                     k_strides=k, v_strides=v, o_strides=o), "flash_window_fwd")
        return s["o"]
    pos = torch.arange(Nk - Nq, Nk, device="cuda")[:, None]
    key = torch.arange(Nk, device="cuda")[None, :]
    seen = key <= pos
    if c["window"]:
        seen = seen & ((pos - key < c["window"]) | (key < c["sinks"]))
    q = s["q"].float().reshape(B, Hkv, (Hq // Hkv) * Nq, d)
    k, v = s["k"].float(), s["v"].float()
    write = None
    if s["lens"] is not None:
        held = key[0][None, :] < s["lens"][:, None]
        v = v.masked_fill(~held[:, None, :, None], 0.0)
        seen = seen[None] & held[:, None, :]
        write = (pos[None, :, 0] < s["lens"][:, None])[:, None, :, None]
        seen = seen[:, None, None]
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"]).view(B, Hkv, Hq // Hkv, Nq, Nk)
    p, total = _weights(scores, seen)
    o = torch.matmul(p.view(B, Hkv, -1, Nk), v).view(B, Hq, Nq, d)
    total = total.view(B, Hq, Nq, 1)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).to(s["o"].dtype)
    return o if write is None else torch.where(write, o, s["o"])


def _exponent(amax):
    """e of the scale 2^e: the smallest with amax <= 448 * 2^e, in [-100, 119]."""
    m, x = torch.frexp(amax)  # amax = m * 2^x, m in [1/2, 1); 448 = 7/8 * 2^9
    e = x - 9 + (m > 0.875).to(x.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, -100)).clamp_(-100, 119)


def _append(s):
    c = s["case"]
    P = c["page"]
    if own:
        from vkcuda_b200 import vc
        vc.check(vc.kv8_append(s["cache"], s["kn"], s["vn"], s["tokens"], s["table"],
                               s["table"].shape[1], s["start"], c["B"], s["most"],
                               vc.Dtype.F16 if c["dtype"] == "fp16" else vc.Dtype.BF16,
                               cu=s["cu"], lens_out=s["lens"]), "kv8_append")
        return [s["k"], s["v"], s["ks"], s["vs"], s["lens"]]
    start = s["start"].long()
    cu = s["cu"].long()
    t = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(cu, t, right=True) - 1
    pos = start[seq] + t - cu[seq]
    page, slot = s["table"][seq, pos // P].long(), pos % P
    # The one page of a sequence that may hold earlier tokens: the page of its first new one.
    kept = start % P
    first = s["table"].gather(1, (start // P).clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0].long()
    row = torch.arange(P, device="cuda")
    old = row[None, :] < kept[:, None]
    for new, codes, scale in ((s["kn"], s["k"], s["ks"]), (s["vn"], s["v"], s["vs"])):
        x = new.float()
        amax = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
        e = torch.full_like(scale, -200.0)
        e[page] = _exponent(amax[page]).float()
        before = torch.log2(scale[first])
        e[first] = torch.where((kept > 0)[:, None], torch.maximum(e[first], before), e[first])
        raw = codes.view(torch.uint8)
        held = raw[first].view(codes.dtype).float()
        moved = (held * torch.exp2(before - e[first])[:, :, None, None]).to(codes.dtype)
        raw[first] = torch.where(old[:, None, :, None], moved.view(torch.uint8), raw[first])
        scale[page] = torch.exp2(e[page])
        raw[page, :, slot] = (x * torch.exp2(-e[page])[:, :, None]).to(codes.dtype).view(torch.uint8)
    torch.add(s["start"], s["cu"][1:] - s["cu"][:-1], out=s["lens"])
    return [s["k"], s["v"], s["ks"], s["vs"], s["lens"]]


def _attn(s):
    c = s["case"]
    B, Hq, Hkv, d, P = (c[k] for k in ("B", "Hq", "Hkv", "d", "page"))
    if own:
        from vkcuda_b200 import vc
        vc.check(vc.kv8_attn(s["cache"], s["q"], s["o"], s["table"], s["table"].shape[1], s["lens"], B, Hq,
                             s["scale"], vc.Dtype.F16 if c["dtype"] == "fp16" else vc.Dtype.BF16, s["ws"],
                             s["ws"].numel(), window=c["window"], sinks=c["sinks"]), "kv8_attn")
        return s["o"]
    ids = s["table"].clamp(min=0).long()
    L = ids.shape[1] * P
    lens = s["lens"][:, None]
    key = torch.arange(L, device="cuda")[None, :]
    seen = key < lens
    if c["window"]:
        seen = seen & ((key >= lens - c["window"]) | (key < c["sinks"]))

    def rows(codes, scale):
        x = codes.view(torch.uint8)[ids].view(codes.dtype).float().mul_(scale[ids][..., None, None])
        x = x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, L, d)
        return x.masked_fill_(~seen[:, None, :, None], 0.0)

    q = s["q"].float().view(B, Hkv, Hq // Hkv, d)
    scores = torch.matmul(q, rows(s["k"], s["ks"]).transpose(-1, -2)).mul_(s["scale"])
    p, total = _weights(scores, seen[:, None, None, :])
    o = torch.matmul(p, rows(s["v"], s["vs"]))
    return torch.where(total > 0, o / total, torch.zeros_like(o)).view(B, Hq, d).to(s["q"].dtype)


def _copy(s):
    if own:
        from vkcuda_b200 import vc
        vc.check(vc.kv8_copy_pages(s["caches"], s["src"], s["dst"], s["src"].numel()), "kv8_copy_pages")
    else:
        src, dst = s["src"].long(), s["dst"].long()
        for x in ("k", "v", "ks", "vs"):
            s[x][:, dst] = s[x][:, src]
    return [s["k"], s["v"], s["ks"], s["vs"]]


# ------------------------------------------------------------------ 64 bits
def _e4m3(x):
    """Nearest e4m3 value (ties to even) of float64 values within +-448: 4 significant bits, steps of
    2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "window":
        B, Hq, Hkv, Nq, Nk, d = (case[k] for k in ("B", "Hq", "Hkv", "Nq", "Nk", "d"))
        if B * Hq * Nq * Nk > 3e9:
            return None
        out = torch.zeros(s["o"].shape, dtype=torch.float64, device="cuda")
        j = torch.arange(Nk, device="cuda")
        for b in range(B):
            n = Nk if s["lens"] is None else int(s["lens"][b])
            last = min(Nq, n - (Nk - Nq))  # rows that belong to the sequence
            if last <= 0:
                continue
            for h in range(Hq):
                k, v = (s[x][b, h // (Hq // Hkv), :n].double() for x in "kv")
                for i0 in range(0, last, 2048):
                    i1 = min(i0 + 2048, last)
                    p = torch.arange(i0, i1, device="cuda") + (Nk - Nq)
                    far = p[:, None] - j[None, :n]
                    hide = far < 0
                    if case["window"]:
                        hide |= (far >= case["window"]) & (j[None, :n] >= case["sinks"])
                    w = (s["q"][b, h, i0:i1].double() @ k.T) / math.sqrt(d)
                    w = torch.softmax(w.masked_fill_(hide, float("-inf")), -1)
                    out[b, h, i0:i1] = torch.nan_to_num(w) @ v
        return out
    if case["op"] == "append":
        P = case["page"]
        got = []
        table, cu, start = s["table"].tolist(), s["cu"].tolist(), s["start"].tolist()
        if sum(len(r) for r in table) > 6000:
            return None
        for new, codes, scale in ((s["kn"], s["k"], s["ks"]), (s["vn"], s["v"], s["vs"])):
            val, sc = codes.double(), scale.double()
            for b in range(case["B"]):
                at, end = start[b], start[b] + cu[b + 1] - cu[b]
                while at < end:
                    n = min(end, (at // P + 1) * P) - at
                    x = new[cu[b] + at - start[b]:cu[b] + at - start[b] + n].double().transpose(0, 1)
                    page, slot = table[b][at // P], at % P
                    top = x.abs().amax((1, 2))
                    # 16-bit inputs lie 2^-12 off a power of two or on it: 1e-9 takes log2's own error.
                    grid = torch.exp2(torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -100)) - 1e-9))
                    if slot:
                        grid = torch.maximum(grid, sc[page])
                        val[page][:, :slot] = _e4m3(val[page][:, :slot] * (sc[page] / grid)[:, None, None])
                    sc[page] = grid
                    val[page][:, slot:slot + n] = _e4m3(x / grid[:, None, None])
                    at += n
            got.append((val, sc))
        return [got[0][0], got[1][0], got[0][1], got[1][1], None]
    if case["op"] == "attn":
        P, Hq, Hkv, d = case["page"], case["Hq"], case["Hkv"], case["d"]
        out = torch.zeros(case["B"], Hq, d, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            i = torch.arange(n, device="cuda")
            if case["window"]:
                i = i[(i >= n - case["window"]) | (i < case["sinks"])]
            page = s["table"][b].long()[i // P]
            for h in range(Hkv):
                k, v = (s[x].view(torch.uint8)[page, h, i % P].view(s[x].dtype).double() * s[x + "s"][page, h].double()[:, None] for x in "kv")
                g = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
                out[b, g] = torch.softmax(s["q"][b, g].double() @ k.T / math.sqrt(d), -1) @ v
        return out
    scales = [s[x].double() for x in ("ks", "vs")]
    for to, of in zip(s["dst"].tolist(), s["src"].tolist()):
        for x in scales:
            x[:, to] = x[:, of]
    return [None, None, *scales]
