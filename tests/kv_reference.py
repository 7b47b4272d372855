"""Plain 64-bit forms of the paged cache's operators, position by position, and random batches."""
import numpy as np
import torch

F64 = torch.float64


class Batch:
    """lens: [(new rows, cached positions before them)]; pages in random order, -1 behind the last."""

    def __init__(self, lens, page, seed, pad=0, spare=3, wide=1):
        rng = np.random.default_rng(seed)
        self.lens, self.page = lens, page
        used = [-(-(n + c) // page) for n, c in lens]
        self.n_pages = sum(used) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), max(used, default=0) + wide), -1, np.int32)
        at = 0
        for i, u in enumerate(used):
            self.table[i, :u] = order[at:at + u]
            at += u
        self.start = np.concatenate([[0], np.cumsum([n for n, _ in lens])]).astype(np.int32)
        self.rows = int(self.start[-1]) + pad
        self.pos0 = np.array([c for _, c in lens], np.int32)

    def device(self, max_new=0):
        from cachepotato_b200.kv import KVBatch
        dev = lambda a: torch.from_numpy(a).cuda()
        return KVBatch(dev(self.start), dev(self.pos0), dev(self.table), rows=self.rows, max_new=max_new)

    def place(self, i, j):
        """(pages, places) of sequence i's positions j."""
        return torch.from_numpy(self.table[i].astype(np.int64))[j // self.page], j % self.page


def pools(b, n_kv, hd, dtype, seed, heads_first=False):
    g = torch.Generator().manual_seed(seed)
    shape = (b.n_pages, n_kv, b.page, hd) if heads_first else (b.n_pages, b.page, n_kv, hd)
    made = [torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2)]
    return [p.transpose(1, 2) for p in made] if heads_first else made


def append(b, q, k, v, kp, vp, gq, gk, eps, R, theta):
    """New (q_out, key pool, value pool) in 64 bits; q_out of rows without a sequence is NaN."""
    out = torch.full(q.shape, float("nan"), dtype=F64)
    kp, vp = kp.cpu().to(F64).clone(), vp.cpu().to(F64).clone()
    freq = torch.tensor([theta ** (-2.0 * j / R) for j in range(R // 2)], dtype=F64)

    def turned(x, gain, pos):
        x = x.cpu().to(F64)
        if gain is not None:
            x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * gain.cpu().to(F64)
        a = pos.to(F64)[:, None, None] * freq
        lo, hi = x[..., :R // 2], x[..., R // 2:R]
        return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), x[..., R:]], -1)

    for i, (n, c) in enumerate(b.lens):
        s = slice(int(b.start[i]), int(b.start[i]) + n)
        pos = torch.arange(c, c + n)
        page, at = b.place(i, pos)
        out[s] = turned(q[s], gq, pos)
        kp[page, at] = turned(k[s], gk, pos)
        vp[page, at] = v[s].cpu().to(F64)
    return out, kp, vp


def attend(b, q, kp, vp, scale, window):
    """(out, bound) in 64 bits: bound is the largest sum of weights times |v| and scores' magnitude per
    row and head, what rounding errors scale with. Rows without a sequence are NaN."""
    rows, H, hd = q.shape
    q, kp, vp = q.to(F64), kp.to(F64), vp.to(F64)
    KV = kp.shape[2]
    out = torch.full(q.shape, float("nan"), dtype=F64, device=q.device)
    size = torch.zeros((rows, H, 1), dtype=F64, device=q.device)
    for i, (n, c) in enumerate(b.lens):
        if n == 0:
            continue
        s = slice(int(b.start[i]), int(b.start[i]) + n)
        j = torch.arange(n + c)
        page, at = (x.to(q.device) for x in b.place(i, j))
        k, v = (p[page, at].permute(1, 0, 2).repeat_interleave(H // KV, 0) for p in (kp, vp))
        z = torch.einsum("thd,hjd->htj", q[s], k) * scale
        p, jj = torch.arange(c, c + n, device=q.device)[:, None], j.to(q.device)[None]
        hidden = (jj > p) | ((jj <= p - window) if window else torch.zeros_like(jj > p))
        z = z.masked_fill(hidden, -torch.inf)
        w = torch.softmax(z, -1)
        v = v.masked_fill((hidden.all(0))[None, :, None], 0.0)
        out[s] = torch.einsum("htj,hjd->thd", w, v)
        size[s] = (torch.einsum("thd,hjd->htj", q[s].abs(), k.abs()).amax(-1) * scale).t()[..., None]
    return out, size
