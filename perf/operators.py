"""What is measured of the paged key/value cache: appending rows (with the head norm and the position
rotation on the way) and attention of new rows over the cached positions.

A batch is ragged: sequence i brings `new` rows (one while it generates, many while its prompt is
read) that stand behind `ctx` cached positions; its pages lie anywhere in the pool.
"""
import math
import random

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    qwen = dict(H=32, KV=4, hd=128)                   # the served model's heads
    return [
        # one generated token of one conversation: latency
        dict(name="append_step", op="append", rows="f32", cache="f32", page=16, heads_first=False, seqs=1, chunks=0,
             new_lo=1, new_hi=1, ctx_lo=512, ctx_hi=512, pad=0, rope=128, norm=True, window=0, lens=1, **qwen),
        # a generation step of 64 sequences, half-size cache
        dict(name="append_step64", op="append", rows="f32", cache="f16", page=16, heads_first=False, seqs=64, chunks=0,
             new_lo=1, new_hi=1, ctx_lo=1, ctx_hi=4096, pad=0, rope=128, norm=True, window=0, lens=2, **qwen),
        # prompts of odd lengths and single tokens in one step: small heads, half of each rotated, no head norm
        dict(name="append_ragged", op="append", rows="bf16", cache="bf16", page=24, heads_first=True, seqs=9, chunks=6,
             new_lo=1, new_hi=301, ctx_lo=0, ctx_hi=2999, pad=5, rope=32, norm=False, window=0, lens=3, H=24, KV=8, hd=64),
        # four prompts of 4096 tokens read in one pass: bandwidth
        dict(name="append_prompts", op="append", rows="bf16", cache="bf16", page=64, heads_first=False, seqs=4, chunks=4,
             new_lo=4096, new_hi=4096, ctx_lo=0, ctx_hi=0, pad=0, rope=128, norm=True, window=0, lens=4, **qwen),
        # one generated token after the benchmark's 512-token prompt
        dict(name="attend_step", op="attend", rows="f32", cache="f32", page=16, heads_first=False, seqs=1, chunks=0,
             new_lo=1, new_hi=1, ctx_lo=512, ctx_hi=512, pad=0, rope=0, norm=False, window=0, lens=5, **qwen),
        # a generation step of 64 conversations of all lengths, f32 rows over a half-size cache
        dict(name="attend_step64", op="attend", rows="f32", cache="f16", page=16, heads_first=False, seqs=64, chunks=0,
             new_lo=1, new_hi=1, ctx_lo=128, ctx_hi=4096, pad=0, rope=0, norm=False, window=0, lens=6, **qwen),
        # one token over a long document
        dict(name="attend_long", op="attend", rows="bf16", cache="bf16", page=64, heads_first=False, seqs=1, chunks=0,
             new_lo=1, new_hi=1, ctx_lo=131071, ctx_hi=131071, pad=0, rope=0, norm=False, window=0, lens=7, **qwen),
        # a large generation step, pages stored head by head
        dict(name="attend_step128", op="attend", rows="bf16", cache="bf16", page=128, heads_first=True, seqs=128, chunks=0,
             new_lo=1, new_hi=1, ctx_lo=1000, ctx_hi=8000, pad=0, rope=0, norm=False, window=0, lens=8, **qwen),
        # the benchmark's 512-token prompt in f32
        dict(name="attend_prompt_f32", op="attend", rows="f32", cache="f32", page=16, heads_first=False, seqs=1, chunks=1,
             new_lo=512, new_hi=512, ctx_lo=0, ctx_hi=0, pad=0, rope=0, norm=False, window=0, lens=9, **qwen),
        # a 4096-token chunk of a long prompt
        dict(name="attend_chunk", op="attend", rows="bf16", cache="bf16", page=64, heads_first=False, seqs=1, chunks=1,
             new_lo=4096, new_hi=4096, ctx_lo=12288, ctx_hi=12288, pad=0, rope=0, norm=False, window=0, lens=10, **qwen),
        # a server's mixed step: one chunk of a prompt beside 47 single tokens
        dict(name="attend_mixed", op="attend", rows="bf16", cache="bf16", page=16, heads_first=False, seqs=48, chunks=1,
             new_lo=2001, new_hi=2001, ctx_lo=500, ctx_hi=8000, pad=3, rope=0, norm=False, window=0, lens=11, **qwen),
        # chunks of odd lengths, seven heads to a cached one, a sliding window
        dict(name="attend_window", op="attend", rows="f16", cache="f16", page=24, heads_first=True, seqs=6, chunks=5,
             new_lo=17, new_hi=1501, ctx_lo=0, ctx_hi=5000, pad=0, rope=0, norm=False, window=1000, lens=12, H=14, KV=2, hd=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hd, KV = rng.choice([64, 128]), rng.choice([1, 2, 4, 8])
    rows, cache = rng.choice([("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16")])
    c = dict(op=rng.choice(["append", "attend", "attend"]), rows=rows, cache=cache, KV=KV,
             H=KV * rng.choice([1, 2, 4, 5, 7, 8] if KV < 8 else [1, 2, 3, 4, 8]), hd=hd,
             page=rng.choice([8, 16, 24, 32, 64, 128, 256]), heads_first=rng.random() < 0.5, pad=rng.choice([0, 0, 1, 7]),
             rope=0, norm=False, window=0, lens=rng.randrange(1 << 30))
    if c["op"] == "append":
        c.update(rope=rng.choice([0, 16, hd // 2, hd, hd]), norm=rng.random() < 0.6)
    elif rng.random() < 0.25:
        c["window"] = _log(rng, 1, 5000)
    kind = rng.choice(["step", "step", "chunk", "mixed"])
    if kind == "step":                                   # single tokens
        n = _log(rng, 1, 200)
        hi = _log(rng, 1, 1000000 // n if n > 8 else 120000)
        c.update(seqs=n, chunks=0, new_lo=1, new_hi=1, ctx_lo=rng.choice([0, hi // 8, hi]), ctx_hi=hi)
    elif kind == "chunk":                                # one to four chunks
        n = rng.randint(1, 4)
        hi = _log(rng, 2, 4096 // n if rows == cache != "f32" else 2048 // n)
        c.update(seqs=n, chunks=n, new_lo=rng.choice([0 if n > 1 else 1, hi // 2, hi]), new_hi=hi, ctx_lo=0, ctx_hi=rng.choice([0, _log(rng, 1, 8000)]))
    else:
        n = _log(rng, 2, 60)
        hi = _log(rng, 2, 1500)
        c.update(seqs=n, chunks=rng.randint(1, 2), new_lo=1, new_hi=hi, ctx_lo=0, ctx_hi=_log(rng, 1, 6000))
    return c


def _lens(case):
    """[(new, ctx)] of the sequences; the chunks stand among the single tokens."""
    rng = random.Random(case["lens"])
    got = [(rng.randint(case["new_lo"], case["new_hi"]) if i < case["chunks"] else 1, rng.randint(case["ctx_lo"], case["ctx_hi"]))
           for i in range(case["seqs"])]
    rng.shuffle(got)
    return got


def work(case):
    lens, H, KV, hd = _lens(case), case["H"], case["KV"], case["hd"]
    T = sum(n for n, _ in lens)
    rs, cs = (4 if case[k] == "f32" else 2 for k in ("rows", "cache"))
    table = 4 * (2 * len(lens) + 1) + 4 * sum(-(-(n + c) // case["page"]) for n, c in lens)
    if case["op"] == "append":
        return {"bytes": T * hd * ((2 * H + 2 * KV) * rs + 2 * KV * cs) + table, "flops": T * hd * (H + KV) * (8 if case["norm"] else 4)}
    w = case["window"] or 1 << 40
    seen = pairs = 0
    for n, c in lens:
        seen += n and n + c - max(0, c - w + 1)
        full = max(0, min(n, w - 1 - c))                 # rows that see everything before them
        pairs += full * c + full * (full + 1) // 2 + (n - full) * min(w, 1 << 40) if n + c > w else n * c + n * (n + 1) // 2
    return {"bytes": 2 * T * H * hd * rs + 2 * seen * KV * hd * cs + table, "flops": 4 * hd * H * pairs}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens, H, KV, hd, P = _lens(case), case["H"], case["KV"], case["hd"], case["page"]
    rt, ct = DT[case["rows"]], DT[case["cache"]]
    T = sum(n for n, _ in lens)
    rows = T + case["pad"]
    used = [-(-(n + c) // P) for n, c in lens]
    n_pages = sum(used) + 3
    wide = max(used) + 1

    def normal(*shape, dtype=rt, scale=1.0):
        return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=g)

    def pool():
        if case["heads_first"]:
            return normal(n_pages, KV, P, hd, dtype=ct).transpose(1, 2)
        return normal(n_pages, P, KV, hd, dtype=ct)

    s = dict(case=case, lens=lens, k_pool=pool(), v_pool=pool())
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu()
    pages = torch.full((len(lens), wide), -1, dtype=torch.int32)
    at, start = 0, [0]
    for i, (n, _) in enumerate(lens):
        pages[i, :used[i]] = order[at:at + used[i]]
        at += used[i]
        start.append(start[-1] + n)
    s["pages"] = pages.cuda()
    s["q_start"] = torch.tensor(start, dtype=torch.int32, device="cuda")
    s["pos0"] = torch.tensor([c for _, c in lens], dtype=torch.int32, device="cuda")
    s["out"] = torch.zeros(rows, H, hd, dtype=rt, device="cuda")
    if case["op"] == "append":
        qkv = normal(rows, H + 2 * KV, hd)               # one projection's output; q, k, v are parts of its rows
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        s["q_norm"], s["k_norm"] = (1 + normal(hd, dtype=torch.float32, scale=0.1) if case["norm"] else None for _ in range(2))
    else:
        s["q"] = normal(rows, H, hd, scale=1.5)
    if own:
        from cachepotato_b200.kv import KVBatch, KVCache
        s["cache"] = KVCache(s["k_pool"], s["v_pool"], rope_dim=case["rope"], rope_theta=1e6)
        s["batch"] = KVBatch(s["q_start"], s["pos0"], s["pages"], rows=rows, max_new=max(n for n, _ in lens))
        s["ws"] = s["cache"].workspace(H)
    return s


def _where(s):
    """Per row: its sequence and its position; the pool's place of every (row's) position."""
    T = s["q_start"][-1:]
    t = torch.arange(s["q"].shape[0], device="cuda")
    live = t < T
    seq = (torch.searchsorted(s["q_start"][1:].contiguous(), t.to(torch.int32), right=True)).clamp(max=len(s["lens"]) - 1)
    return live, seq, s["pos0"][seq] + t - s["q_start"][seq]


def _norm(x, gain):
    return x if gain is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * gain


def _rotate(x, pos, R):
    if not R:
        return x
    j = torch.arange(R // 2, dtype=torch.float64, device="cuda")
    a = pos.to(torch.float64)[:, None, None] * 1e6 ** (-2.0 * j / R)
    cos, sin = a.cos().float(), a.sin().float()
    lo, hi, rest = x[..., :R // 2], x[..., R // 2:R], x[..., R:]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, rest], -1)


def _append(s):
    P, R = s["case"]["page"], s["case"]["rope"]
    live, seq, pos = _where(s)
    live = live.nonzero()[:, 0]
    seq, pos = seq[live], pos[live]
    s["out"][live] = _rotate(_norm(s["q"][live].float(), s["q_norm"]), pos, R).to(s["out"].dtype)
    page = s["pages"][seq, pos // P].long()
    s["k_pool"][page, pos % P] = _rotate(_norm(s["k"][live].float(), s["k_norm"]), pos, R).to(s["k_pool"].dtype)
    s["v_pool"][page, pos % P] = s["v"][live].to(s["v_pool"].dtype)
    return [s["out"], s["k_pool"], s["v_pool"]]


def _gather(s, i, n):
    """Keys and values of sequences i (a range or a tensor) at positions 0..n-1, in 32 bits: (len(i), KV, n, hd)."""
    P = s["case"]["page"]
    j = torch.arange(n, device="cuda")
    page = s["pages"][i][:, j // P].clamp(min=0).long()
    return (p[page, j % P].float().transpose(1, 2) for p in (s["k_pool"], s["v_pool"]))


def _softmax_av(q, k, v, pos, window):
    """q (b, KV, G, n, hd) at positions pos (b, n) over k, v (b, KV, len, hd)."""
    x = (q * q.shape[-1] ** -0.5) @ k[:, :, None].transpose(-1, -2)
    j = torch.arange(k.shape[2], device="cuda")
    hidden = j > pos[..., None]
    if window:
        hidden = hidden | (j <= pos[..., None] - window)
    x.masked_fill_(hidden[:, None, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    return (x @ v[:, :, None]) / x.sum(-1, keepdim=True)


def _attend_singles(s, i):
    """All sequences with one new row, as one padded batch."""
    c = s["case"]
    at = s["q_start"][i].long()
    k, v = _gather(s, i, max(s["lens"][x][1] + 1 for x in i.tolist()))
    j = torch.arange(k.shape[2], device="cuda")
    v = v.masked_fill((j > s["pos0"][i][:, None])[:, None, :, None], 0.0)
    q = s["q"][at].float().view(len(at), c["KV"], c["H"] // c["KV"], 1, c["hd"])
    s["out"][at] = _softmax_av(q, k, v, s["pos0"][i][:, None], c["window"]).view(len(at), c["H"], c["hd"]).to(s["out"].dtype)


def _attend_chunk(s, i, at, head):
    """One sequence's chunk, the query heads of one cached head."""
    c, (n, ctx) = s["case"], s["lens"][i]
    G = c["H"] // c["KV"]
    k, v = (x[:, head:head + 1] for x in _gather(s, slice(i, i + 1), n + ctx))
    q = s["q"][at:at + n, head * G:head * G + G].float().transpose(0, 1)[None, None]
    pos = ctx + torch.arange(n, device="cuda")[None]
    s["out"][at:at + n, head * G:head * G + G] = _softmax_av(q, k, v, pos, c["window"])[0, 0].transpose(0, 1).to(s["out"].dtype)


def _attend(s):
    lens, KV = s["lens"], s["case"]["KV"]
    singles = [i for i, (n, _) in enumerate(lens) if n == 1]
    starts = [sum(n for n, _ in lens[:i]) for i in range(len(lens))]
    if singles:
        _attend_singles(s, torch.tensor(singles))
    [_attend_chunk(s, i, starts[i], h) for i, (n, _) in enumerate(lens) if n > 1 for h in range(KV)]
    return s["out"]


def run(s):
    c = s["case"]
    if own:
        if c["op"] == "append":
            s["cache"].append(s["batch"], s["q"], s["k"], s["v"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, q_out=s["out"])
            return [s["out"], s["k_pool"], s["v_pool"]]
        return s["cache"].attend(s["batch"], s["q"], window=c["window"], out=s["out"], ws=s["ws"])
    return _append(s) if c["op"] == "append" else _attend(s)


def exact(case, seed):
    """The definition, row by row of the batch, in 64 bits: complex rotation, weights from the log of the sum."""
    s = prepare(case, seed)
    lens, H, KV, hd, P = s["lens"], case["H"], case["KV"], case["hd"], case["page"]
    G = H // KV
    out = s["out"].double()
    kp, vp = s["k_pool"], s["v_pool"]
    if case["op"] == "append":
        kp, vp = kp.double(), vp.double()
    row = 0
    for i, (n, ctx) in enumerate(lens):
        if not n:
            continue
        pos = torch.arange(ctx, ctx + n, device="cuda")
        if case["op"] == "append":
            def turned(x, gain):
                x = x[row:row + n].double()
                if gain is not None:
                    x = x / (x.pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * gain.double()
                R = case["rope"]
                if R:
                    f = torch.exp(torch.arange(0, R, 2, dtype=torch.float64, device="cuda") * (-math.log(1e6) / R))
                    turn = torch.polar(torch.ones(n, R // 2, dtype=torch.float64, device="cuda"), pos.double()[:, None] * f)
                    z = torch.complex(x[..., :R // 2].contiguous(), x[..., R // 2:R].contiguous()) * turn[:, None]
                    x = torch.cat([z.real, z.imag, x[..., R:]], -1)
                return x
            out[row:row + n] = turned(s["q"], s["q_norm"])
            page = s["pages"][i, (pos // P)].long()
            kp[page, pos % P] = turned(s["k"], s["k_norm"])
            vp[page, pos % P] = s["v"][row:row + n].double()
        else:
            j = torch.arange(n + ctx, device="cuda")
            page = s["pages"][i, j // P].long()
            bias = torch.zeros(n, n + ctx, dtype=torch.float64, device="cuda")
            bias[j[None] > pos[:, None]] = -math.inf
            if case["window"]:
                bias[pos[:, None] - j[None] >= case["window"]] = -math.inf
            for h in range(KV):
                k, v = (p[page, j % P, h].double() for p in (kp, vp))
                for g in range(h * G, h * G + G):
                    z = torch.addmm(bias, s["q"][row:row + n, g].double(), k.t(), alpha=1.0 / math.sqrt(hd))
                    out[row:row + n, g] = (z - torch.logsumexp(z, -1, keepdim=True)).exp_() @ v
        row += n
    return [out, kp, vp] if case["op"] == "append" else out
