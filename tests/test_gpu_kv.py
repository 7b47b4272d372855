"""The paged key/value cache (cpg_kv_append, cpg_kv_attend) against plain 64-bit forms.

Tolerances, with u = 2^-24 (half a step of f32) and e = finfo.eps / 2 of the rows' or the cache's type:
append: an f32 chain of fewer than 32 roundings (a sum of squares of depth 12, division, root, two
  gains, two products and a sum of the rotation; the angle's 2^-25 half turns are 3.2 u), relative to
  the rotated pair's length, and the one rounding to the output's type.
attend: scores carry 16 u of scale·sum|q k| (operand terms of 22 bits, eight sums of 16 products),
  the exponential 4 u; an average with relative weight errors d is off by at most 2 d max|v|; the
  running sums add one rounding per 16 positions. 16-bit rows: each weight is off by e besides (at
  most 2 e max|v| of the average, weights and their sum), and the result by e of itself."""
import ctypes

import numpy as np
import pytest
import torch

import kv_reference as R
from cachepotato_b200._lib import CpgError

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
COMBOS = [("f32", "f32"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step among the type's subnormals, where a rounding is not relative to the value."""
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


def rows(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def close(got, want, tol, what):
    got, tol = got.double().cpu(), torch.as_tensor(tol).double().cpu().expand(want.shape)
    want = want.cpu()
    live = ~torch.isnan(want)
    off = ((got - want).abs() / tol)[live]
    assert torch.isfinite(got[live]).all(), what
    assert off.numel() == 0 or off.max() <= 1, f"{what}: {float(off.max()):.3g} times the tolerance"


# ------------------------------------------------------------------------------------------ append
def check_append(lens, page, H, KV, hd, rt, ct, rope, norm, heads_first=False, pad=0, theta=1e6, seed=0, inplace=False,
                 fused=True):
    from cachepotato_b200.kv import KVCache
    b = R.Batch(lens, page, seed, pad=pad)
    kp, vp = R.pools(b, KV, hd, ct, seed + 1, heads_first)
    if fused:
        qkv = rows((b.rows, H + 2 * KV, hd), rt, seed + 2)
        q, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    else:
        q, k, v = rows((b.rows, H, hd), rt, seed + 2), rows((b.rows, KV, hd), rt, seed + 3), rows((b.rows, KV, hd), rt, seed + 4)
    gq, gk = ((1 + 0.1 * rows((hd,), torch.float32, seed + 5 + i)) if norm else None for i in range(2))
    want = R.append(b, q.cpu(), k.cpu(), v.cpu(), kp, vp, gq, gk, 1e-6, rope, theta)
    cache = KVCache(kp, vp, rope_dim=rope, rope_theta=theta)
    q_in = q.clone()
    before = q_in if inplace else torch.full_like(q_in, 7.0)
    out = cache.append(b.device(), q_in if inplace else q, k, v, q_norm=gq, k_norm=gk, q_out=before)
    cache.check()
    assert out is before

    def tol(w, dtype):
        amp = w.abs().clone()
        amp[..., :rope] = torch.hypot(w[..., :rope], torch.cat([w[..., rope // 2:rope], w[..., :rope // 2]], -1))
        return half_step(dtype) * w.abs() * (1 + 2 ** -8) + 32 * U * amp + tiny(dtype)
    close(out, want[0], tol(want[0], rt), "q")
    close(kp, want[1], tol(want[1], ct), "keys")
    close(vp, want[2], half_step(ct) * want[2].abs() + tiny(ct), "values")
    # rows of no sequence and pages of no new row: untouched
    T = int(b.start[-1])
    assert torch.equal(out[T:], q[T:] if inplace else torch.full_like(q[T:], 7.0))


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("hd", [64, 128])
def test_append_types(rt, ct, hd):
    check_append([(1, 0), (3, 15), (0, 40), (17, 31), (1, 700)], 16, 8, 2, hd, TYPES[rt], TYPES[ct], hd, True, pad=3)


@pytest.mark.parametrize("rope", [0, 16, 32, 64, 128])
@pytest.mark.parametrize("norm", [False, True])
def test_append_rotated_part(rope, norm):
    check_append([(5, 3), (1, 64)], 8, 6, 3, 128, torch.float32, torch.bfloat16, rope, norm, heads_first=True, fused=False)


@pytest.mark.parametrize("H,KV", [(1, 1), (32, 4), (14, 2), (64, 8), (5, 5)])
def test_append_heads_and_in_place(H, KV):
    check_append([(1, 9)], 24, H, KV, 128, torch.bfloat16, torch.bfloat16, 128, True, inplace=True)
    check_append([(211, 9), (90, 0)], 24, H, KV, 64, torch.float32, torch.float16, 32, True, inplace=True, pad=1)


def test_append_far_positions():
    """Positions past two million: an f32 angle would be off by 0.1."""
    page = 65536
    b = R.Batch([(2, 2_000_003), (1, 31)], page, 1)
    b.n_pages = 3
    b.table = np.full((2, 32), -1, np.int32)
    b.table[0, 2_000_003 // page], b.table[1, 0] = 2, 0
    from cachepotato_b200.kv import KVCache
    kp, vp = R.pools(b, 1, 64, torch.float32, 2)
    q, k, v = (rows((3, 1, 64), torch.float32, 3 + i) for i in range(3))
    want = R.append(b, q.cpu(), k.cpu(), v.cpu(), kp, vp, None, None, 0.0, 64, 1e4)
    out = KVCache(kp, vp, rope_dim=64, rope_theta=1e4).append(b.device(), q, k, v)
    amp = torch.hypot(want[0], torch.cat([want[0][..., 32:], want[0][..., :32]], -1))
    close(out, want[0], 32 * U * amp, "q")
    assert torch.isfinite(kp).all()
    page_at = 2_000_003 % page
    close(kp[2, page_at:page_at + 2], want[1][2, page_at:page_at + 2], 64 * U, "keys")


def test_append_many_sequences_and_lookup():
    """Rows find their sequence among many, empty ones between them."""
    rng = np.random.default_rng(5)
    for n in (31, 33, 34, 700, 1100):
        lens = [(int(x), int(c)) for x, c in zip(rng.integers(0, 3, n), rng.integers(0, 20, n))]
        check_append(lens, 8, 2, 1, 64, torch.float32, torch.float32, 64, False, seed=n, pad=2)


def test_append_without_queries_and_reference_angles():
    from cachepotato_b200.kv import KVCache
    b = R.Batch([(4, 500)], 16, 9)
    kp, vp = R.pools(b, 2, 128, torch.float32, 10)
    k, v = rows((4, 2, 128), torch.float32, 11), rows((4, 2, 128), torch.float32, 12)
    cache = KVCache(kp, vp, rope_theta=1e6, rope_f32=True)
    assert cache.append(b.device(), None, k, v) is None
    cache.check()
    page, at = b.place(0, torch.arange(500, 504))
    got = kp[page.cuda(), at.cuda()].cpu()
    inv = np.float32(1e6) ** (np.arange(64, dtype=np.float32) * np.float32(-2.0) / np.float32(128.0))
    ang = (np.arange(500, 504, dtype=np.float32)[:, None, None] * inv).astype(np.float32)   # the reference's f32 angle
    c, s = np.cos(ang.astype(np.float64)), np.sin(ang.astype(np.float64))
    x = k.cpu().double().numpy()
    want = np.concatenate([x[..., :64] * c - x[..., 64:] * s, x[..., 64:] * c + x[..., :64] * s], -1)
    # powf may differ from the host's by 4 steps of the frequency: 4 · 2^-23 · 504 of the angle
    amp = np.hypot(x[..., :64], x[..., 64:])
    assert np.all(np.abs(got.numpy() - want) <= (8 * U * ang.max() + 32 * U) * np.concatenate([amp, amp], -1))


# ------------------------------------------------------------------------------------------ attend
def check_attend(lens, page, H, KV, hd, rt, ct, heads_first=False, pad=0, window=0, seed=0, scale=None, max_new=None, ws=None,
                 q_scale=1.5):
    from cachepotato_b200.kv import KVCache
    b = R.Batch(lens, page, seed, pad=pad)
    kp, vp = R.pools(b, KV, hd, ct, seed + 1, heads_first)
    poison(b, kp, vp)
    q = rows((b.rows, H, hd), rt, seed + 2, q_scale)
    scale_ = hd ** -0.5 if scale is None else scale
    want, size = R.attend(b, q, kp, vp, scale_, window)
    cache = KVCache(kp, vp, rope_dim=0)
    out = torch.full_like(q, 7.0)
    most = max((n for n, _ in lens), default=0)
    got = cache.attend(b.device(most if max_new is None else max_new), q, scale=scale, window=window, out=out, ws=ws)
    cache.check()
    assert got is out
    close(got, want, attend_tol(b, want, size, vp, rt), f"{lens[:4]}")
    T = int(b.start[-1])
    assert bool((got[T:] == 7.0).all())


def poison(b, kp, vp):
    """Everything no row may look at holds NaN or infinities: pages of nobody, places behind a sequence's end."""
    free = torch.ones(b.n_pages, b.page, dtype=torch.bool)
    for i, (n, c) in enumerate(b.lens):
        if n:
            page, at = b.place(i, torch.arange(n + c))
            free[page, at] = False
    free = free.cuda()
    kp[free] = float("nan")
    vp[free] = float("inf")


def attend_tol(b, want, size, vp, rt):
    v = vp[torch.isfinite(vp)].abs().max().double() if vp.numel() else 1.0
    n = max((n + c for n, c in b.lens), default=1)
    tol = (2 * (16 * size + 4) + n / 16 + 32) * U * v
    if rt != torch.float32:
        tol = tol + half_step(rt) * (2 * v + want.abs()) + tiny(rt) * (1 + n * v)
    return tol.expand(want.shape)


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("heads_first", [False, True])
def test_attend_single_rows(rt, ct, hd, heads_first):
    lens = [(1, 0), (1, 1), (0, 9), (1, 15), (1, 16), (1, 62), (1, 63), (1, 64), (1, 130), (1, 1000), (1, 517)]
    check_attend(lens, 16, 8, 2, hd, TYPES[rt], TYPES[ct], heads_first, pad=2)


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("hd", [64, 128])
def test_attend_chunks(rt, ct, hd):
    lens = [(2, 0), (129, 3), (1, 77), (64, 0), (0, 5), (33, 500), (300, 129)]
    check_attend(lens, 24, 8, 2, hd, TYPES[rt], TYPES[ct], pad=3)


@pytest.mark.parametrize("H,KV", [(1, 1), (4, 4), (14, 2), (10, 2), (32, 4), (16, 1), (34, 2), (40, 1)])
@pytest.mark.parametrize("rt,ct", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_attend_head_groups(H, KV, rt, ct):
    check_attend([(1, 200), (1, 33)], 32, H, KV, 128, TYPES[rt], TYPES[ct])
    check_attend([(37, 91), (1, 300), (150, 0)], 32, H, KV, 64, TYPES[rt], TYPES[ct], heads_first=True)


@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 72, 128, 200, 256, 384])
@pytest.mark.parametrize("rt,ct", [("f32", "f32"), ("bf16", "bf16")])
def test_attend_pages(page, rt, ct):
    """Pages that end inside a tile, and tiles inside a page."""
    check_attend([(1, 333), (140, 250), (1, 0)], page, 8, 1, 128, TYPES[rt], TYPES[ct])
    check_attend([(1, 333), (1, 130)], page, 8, 1, 128, TYPES[rt], TYPES[ct])


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 128, 1000])
@pytest.mark.parametrize("rt,ct", [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
def test_attend_window(window, rt, ct):
    check_attend([(1, 5), (1, 400), (1, 63)], 16, 8, 2, 64, TYPES[rt], TYPES[ct], window=window)
    check_attend([(70, 300), (1, 400), (200, 0)], 16, 8, 2, 128, TYPES[rt], TYPES[ct], window=window)


@pytest.mark.parametrize("max_new", [0, 1, 2, 1000])
@pytest.mark.parametrize("rt,ct", [("f32", "f32"), ("bf16", "bf16")])
def test_attend_any_hint(max_new, rt, ct):
    """max_new only chooses the kernel."""
    check_attend([(1, 100), (90, 41), (3, 7)], 16, 8, 2, 128, TYPES[rt], TYPES[ct], max_new=max_new)


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("window", [0, 100])
def test_attend_chunks_beside_single_rows(rt, ct, window):
    """A step's single tokens and prompt chunks, lengths on both sides of every choice of kernel between
    them, empty sequences, more sequences than a block has threads; any hint gives the same rows."""
    rng = np.random.default_rng(17)
    some = [(1, int(c)) for c in rng.integers(0, 600, 20)]
    check_attend(some[:9] + [(200, 333)] + some[9:] + [(0, 9), (3, 50)], 16, 8, 2, 128, TYPES[rt], TYPES[ct], window=window, pad=2)
    check_attend(some + [(8, 40), (9, 40), (7, 0), (64, 5), (4, 1), (5, 90)], 24, 16, 4, 64, TYPES[rt], TYPES[ct], window=window)
    many = [(int(n), int(c)) for n, c in zip(rng.integers(0, 3, 450), rng.integers(0, 60, 450))]
    many[7], many[440] = (150, 20), (33, 70)
    for max_new in (150, 1, 0):
        check_attend(many, 8, 4, 2, 64, TYPES[rt], TYPES[ct], window=window, max_new=max_new)


@pytest.mark.parametrize("rt,ct", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
def test_attend_long_and_many(rt, ct):
    check_attend([(1, 20011)], 64, 8, 1, 128, TYPES[rt], TYPES[ct])
    rng = np.random.default_rng(3)
    check_attend([(1, int(c)) for c in rng.integers(0, 900, 300)], 16, 4, 2, 64, TYPES[rt], TYPES[ct])
    check_attend([(int(n), int(c)) for n, c in zip(rng.integers(0, 40, 150), rng.integers(0, 300, 150))], 16, 4, 2, 64,
                 TYPES[rt], TYPES[ct])


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("new", [1, 150])
def test_attend_needles(rt, ct, new):
    """One key per row outweighs all others (score 60 above them): just inside and just outside of what
    the row sees, at the window's edge and at its own position. Wrong masks change the result by the
    needle's whole value, whatever the type's rounding."""
    from cachepotato_b200.kv import KVCache
    hd, ctx, window = 64, 333, 100
    b = R.Batch([(new, ctx)], 16, 4)
    for edge in (0, 1, -(window - 1), -window):                   # j = p + edge
        kp, vp = R.pools(b, 1, hd, TYPES[ct], 5)
        t = new - 1 if new == 1 else 77                           # the row under test
        p = ctx + t
        kp.mul_(0.01)
        q = rows((new, 2, hd), TYPES[rt], 6, 0.01)
        q[t] = 0.0
        q[t, :, 3] = 60.0
        page, at = b.place(0, torch.tensor([p + edge]))
        if page[0] < 0 or p + edge >= new + ctx:
            continue
        kp[page.cuda(), at.cuda(), 0, 3] = 8.0
        want, size = R.attend(b, q, kp, vp, hd ** -0.5, window)
        got = KVCache(kp, vp, rope_dim=0).attend(b.device(new), q, window=window)
        close(got, want, attend_tol(b, want, size, vp, TYPES[rt]), f"edge {edge}")
        at_needle = vp[page.cuda(), at.cuda(), 0][0].double()
        seen = edge in (0, -(window - 1))
        assert bool(torch.allclose(got[t, 0].double(), at_needle, atol=0.05)) == seen, edge


@pytest.mark.parametrize("rt,ct", COMBOS)
def test_attend_scores_of_any_size(rt, ct):
    """Scores in the thousands, rising along the cache (the running maximum moves at every tile), of
    one sign, and all equal."""
    from cachepotato_b200.kv import KVCache
    hd = 128
    for kind in ("rising", "falling", "equal", "huge"):
        b = R.Batch([(1, 700), (40, 600)], 16, 8)
        kp, vp = R.pools(b, 1, hd, TYPES[ct], 9)
        q = rows((b.rows, 8, hd), TYPES[rt], 10, 0.01)
        q[..., 0] = 8.0
        for i, (n, c) in enumerate(b.lens):
            j = torch.arange(n + c)
            page, at = (x.cuda() for x in b.place(i, j))
            ramp = {"rising": j * 0.25, "falling": 100 - j * 0.25, "equal": j * 0.0, "huge": (j % 7) * 500.0}[kind]
            kp[page, at, 0] = 0.0 if kind == "equal" else 0.01
            kp[page, at, 0, 0] = ramp.to(TYPES[ct]).cuda()
        want, size = R.attend(b, q, kp, vp, hd ** -0.5, 0)
        got = KVCache(kp, vp, rope_dim=0).attend(b.device(40), q)
        # the score's own scale enters its error: 16 u of up to 2000
        close(got, want, attend_tol(b, want, size, vp, TYPES[rt]), kind)


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("new", [1, 40])
def test_attend_many_small_weights(rt, ct, new):
    """A few keys at the start outweigh each of the others by far, and all of them together not at all:
    thousands of equal weights of 2^-15 to 2^-26 of the largest. Values are positive, so what each weight is
    off by adds up, and is relative to the result: attend_tol's parts, a half step of a 16-bit weight (and one of the result), and
    2^-25 of a lifted f16 one, the largest of which is over 2^6 (so 2^-31 each). 300 sequences over the same pages: a block then works through most of one, with the
    large keys in front, where a lone sequence would be spread over all blocks."""
    from cachepotato_b200.kv import KVBatch, KVCache
    hd, H, S = 64, 4, 300
    for n, below in ((4000, 10.5), (4000, 17.4), (131000, 10.0), (131000, 14.1), (131000, 17.4), (131000, 18.0)):
        b = R.Batch([(new, n)], 256, 8)
        kp, vp = R.pools(b, 1, hd, TYPES[ct], 9)
        vp.copy_((1 + 0.1 * vp.float()).to(TYPES[ct]))
        q = torch.zeros((new, H, hd), dtype=TYPES[rt], device="cuda")
        q[..., 0] = 8.0
        kp.zero_()
        page, at = (x.cuda() for x in b.place(0, torch.arange(0, 64, 16)))
        kp[page, at, 0, 0] = below                                # a score of `below`; the others' are 0
        vp[page, at] = 0.25
        want, size = R.attend(b, q, kp, vp, hd ** -0.5, 0)
        tol = (2 * (16 * size + 4) + (n + new) / 16 + 32) * U * want
        if rt != "f32":
            tol = tol + half_step(TYPES[rt]) * 2 * want * (1 + 2 ** -7) + n * 2.0 ** -31 * vp.max().double()
        i32 = dict(dtype=torch.int32, device="cuda")
        batch = KVBatch(torch.arange(S + 1, **i32) * new, torch.full((S,), n, **i32),
                        torch.from_numpy(b.table).cuda().repeat(S, 1), rows=S * new, max_new=new)
        got = KVCache(kp, vp, rope_dim=0).attend(batch, q.repeat(S, 1, 1))
        close(got, want.repeat(S, 1, 1), tol.expand(want.shape).repeat(S, 1, 1), f"{n}, {below}")


@pytest.mark.parametrize("rt,ct", [c for c in COMBOS if c[0] == "f32"])
@pytest.mark.parametrize("new", [1, 90])
@pytest.mark.parametrize("hd", [64, 128])
def test_attend_rows_with_one_large_element(rt, ct, new, hd):
    """f32 rows keep their precision beside an element that is 30000 times as large and meets zeros."""
    from cachepotato_b200.kv import KVCache
    for big in (30000.0, -1.2e-30, 0.0):                          # the rest is scaled like it: 1, 4e-35, and plain
        b = R.Batch([(new, 20), (new, 3)], 16, 8)
        kp, vp = R.pools(b, 1, hd, TYPES[ct], 9)
        q = rows((b.rows, 8, hd), torch.float32, 10)
        scale = hd ** -0.5
        if big:
            kp[..., 5] = 0.0
            q.mul_(abs(big) / 30000)
            scale *= 30000 / abs(big)
            q[..., 5] = big
        want, size = R.attend(b, q, kp, vp, scale, 0)
        got = KVCache(kp, vp, rope_dim=0).attend(b.device(new), q, scale=scale)
        close(got, want, attend_tol(b, want, size, vp, torch.float32), f"{big}")


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("new", [1, 90])
def test_attend_rows_of_zeros_and_small_scales(rt, ct, new):
    """Rows of zeros among others, and a scale that makes all weights equal."""
    from cachepotato_b200.kv import KVCache
    for scale in (0.125, 1e-9, 1e-37):
        b = R.Batch([(new, 20), (new, 3)], 16, 8)
        kp, vp = R.pools(b, 1, 64, TYPES[ct], 9)
        q = rows((b.rows, 8, 64), TYPES[rt], 10)
        q[::2] = 0.0
        want, size = R.attend(b, q, kp, vp, scale, 0)
        got = KVCache(kp, vp, rope_dim=0).attend(b.device(new), q, scale=scale)
        close(got, want, attend_tol(b, want, size, vp, TYPES[rt]), f"scale {scale}")


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 40])
def test_attend_counts_every_position_once(rt, ct, hd, new):
    """Equal weights over values that tell which run of 16 positions they come from: each output counts the
    positions of some runs. Weights and sums are exact, so what remains is the division (4 u) and the
    result's own rounding; a run lost or added twice is off by some part of a fifth."""
    from cachepotato_b200.kv import KVCache
    for window in (0, 1000):
        b = R.Batch([(new, 5000), (1, 77), (new, 1311), (new, 16 * hd - 1), (0, 4)], 24, 5)
        kp, vp = R.pools(b, 2, hd, TYPES[ct], 6)
        vp.zero_()
        for i, (n, c) in enumerate(b.lens):
            if n:
                j = torch.arange(n + c)
                page, at = b.place(i, j)
                vp[page.cuda(), at.cuda(), :, (j // 16 % hd).cuda()] = 1.0
        q = torch.zeros((b.rows, 8, hd), dtype=TYPES[rt], device="cuda")
        want, _ = R.attend(b, q, kp, vp, hd ** -0.5, window)
        got = KVCache(kp, vp, rope_dim=0).attend(b.device(new), q, window=window)
        off = 4 * U if rt == "f32" else half_step(TYPES[rt]) * (1 + 2 ** -7)
        close(got, want, off * want + tiny(TYPES[rt]), f"window {window}")


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("new", [1, 80])
def test_one_page_many_times(rt, ct, new):
    """Many cached heads over a long table that names the same page again and again: what a row sees is that
    page's positions over and over, so the result is the page's own."""
    from cachepotato_b200.kv import KVBatch, KVCache
    page, KV, hd, times = 64, 128 if new == 1 else 16, 64, 1500
    one = R.Batch([(1, page - 1)], page, 3, spare=0)
    kp, vp = R.pools(one, KV, hd, TYPES[ct], 4)
    q = rows((1, 2 * KV, hd), TYPES[rt], 5).repeat(new, 1, 1)
    want, size = R.attend(one, q[:1], kp, vp, hd ** -0.5, 0)
    i32 = dict(dtype=torch.int32, device="cuda")
    arrays = (torch.arange(new + 1, **i32), torch.full((new,), page * times - 1, **i32), torch.zeros((new, times), **i32))
    cache = KVCache(kp, vp, rope_dim=0)
    tol = attend_tol(R.Batch([(1, page * times)], page, 3), want, size, vp, TYPES[rt])
    for hint in (1, 80):                                          # single rows on both kinds of kernel
        got = cache.attend(KVBatch(*arrays, rows=new, max_new=hint), q)
        cache.check()
        close(got, want.repeat(new, 1, 1), tol.repeat(new, 1, 1), f"hint {hint}")


def test_attend_scale_and_in_place():
    from cachepotato_b200.kv import KVCache
    for rt, ct in COMBOS:
        check_attend([(1, 90), (50, 10)], 16, 4, 1, 64, TYPES[rt], TYPES[ct], scale=0.5)
        b = R.Batch([(1, 90), (50, 10)], 16, 3)
        kp, vp = R.pools(b, 1, 64, TYPES[ct], 4)
        cache, q = KVCache(kp, vp, rope_dim=0), rows((51, 4, 64), TYPES[rt], 5)
        want = cache.attend(b.device(50), q)
        assert cache.attend(b.device(50), q, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("new", [1, 100])
def test_pages_in_front_of_the_window_may_be_gone(rt, ct, new):
    """Positions no row sees any more are not looked up: their table entries may be anything."""
    from cachepotato_b200.kv import KVCache
    window, page = 70, 16
    b = R.Batch([(new, 500), (new, 3)], page, 6)
    kp, vp = R.pools(b, 2, 128, TYPES[ct], 7)
    q = rows((b.rows, 8, 128), TYPES[rt], 8)
    cache, batch = KVCache(kp, vp, rope_dim=0), b.device(new)
    want = cache.attend(batch, q, window=window)
    gone = (500 - window + 1) // page                             # pages that end before the first row's window
    batch.pages[0, :gone] = torch.tensor([-1, b.n_pages, -7] * gone, dtype=torch.int32, device="cuda")[:gone]
    assert torch.equal(cache.attend(batch, q, window=window), want)
    cache.check()


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("hd", [64, 128])
def test_places_in_front_of_the_window_may_hold_anything(rt, ct, new, page, hd):
    """A caller that writes only the positions some row sees: every place in front of the first row's
    window holds NaN and infinities, those of a page that is still read among them."""
    from cachepotato_b200.kv import KVCache
    for window in (1, 33, 70):
        b = R.Batch([(new, 500), (new, 3), (new, 117)], page, 6)
        kp, vp = R.pools(b, 2, hd, TYPES[ct], 7)
        q = rows((b.rows, 8, hd), TYPES[rt], 8)
        want, size = R.attend(b, q, kp, vp, hd ** -0.5, window)
        tol = attend_tol(b, want, size, vp, TYPES[rt])
        for i, (_, c) in enumerate(b.lens):
            at = b.place(i, torch.arange(max(0, c - window + 1)))
            page_at, place = (x.cuda() for x in at)
            kp[page_at, place] = float("nan")
            vp[page_at, place] = torch.tensor([float("inf"), float("nan"), -float("inf"), float("nan")], dtype=TYPES[ct],
                                              device="cuda").repeat(hd // 4)
        cache = KVCache(kp, vp, rope_dim=0)
        close(cache.attend(b.device(new), q, window=window), want, tol, f"window {window}")
        cache.check()


@pytest.mark.parametrize("rt,ct", COMBOS)
def test_one_pool_for_keys_and_values(rt, ct):
    """Keys and values side by side in one tensor, part of a wider one: strides of no dense layout."""
    from cachepotato_b200.kv import KVCache
    b = R.Batch([(1, 90), (40, 33), (0, 4), (1, 0)], 16, 3, pad=1)
    big = torch.full((b.n_pages, 3, 16, 4, 2, 64), 9.0, dtype=TYPES[ct], device="cuda")
    kp, vp = big[:, 0, :, 1:3, 0], big[:, 2, :, 1:3, 0]           # (pages, places, 2 of 4 heads, 64)
    for p, s in ((kp, 4), (vp, 5)):
        p.copy_(rows(p.shape, TYPES[ct], s))
    rest = torch.ones_like(big, dtype=torch.bool)
    rest[:, 0, :, 1:3, 0] = rest[:, 2, :, 1:3, 0] = False
    qkv = rows((b.rows, 12, 64), TYPES[rt], 6)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    cache = KVCache(kp, vp, rope_theta=1e4)
    want = R.append(b, q.cpu(), k.cpu(), v.cpu(), kp, vp, None, None, 0.0, 64, 1e4)
    qr = cache.append(b.device(40), q, k, v)
    amp = lambda w: torch.hypot(w, torch.cat([w[..., 32:], w[..., :32]], -1))
    close(kp, want[1], half_step(TYPES[ct]) * want[1].abs() * (1 + 2 ** -8) + 32 * U * amp(want[1]) + tiny(TYPES[ct]), "keys")
    close(vp, want[2], half_step(TYPES[ct]) * want[2].abs() + tiny(TYPES[ct]), "values")
    assert bool((big[rest] == 9.0).all())
    qr[int(b.start[-1]):] = 0
    ref, size = R.attend(b, qr, kp, vp, 64 ** -0.5, 0)
    close(cache.attend(b.device(40), qr), ref, attend_tol(b, ref, size, vp, TYPES[rt]), "attend")
    cache.check()


@pytest.mark.parametrize("H,KV", [(100, 1), (130, 1), (256, 2)])
@pytest.mark.parametrize("rt,ct", [("f32", "f16"), ("bf16", "bf16")])
def test_attend_very_many_heads_to_a_cached_one(H, KV, rt, ct):
    check_attend([(1, 200), (9, 33), (3, 0)], 16, H, KV, 64, TYPES[rt], TYPES[ct], max_new=9)


@pytest.mark.parametrize("rt,ct", [("f32", "f32"), ("bf16", "bf16")])
def test_rows_in_front_of_the_first_sequence(rt, ct):
    """q_start need not begin at zero: earlier rows belong to nobody."""
    from cachepotato_b200.kv import KVBatch, KVCache
    for new in (1, 60):
        b = R.Batch([(new, 20), (1, 70)], 16, 3)
        kp, vp = R.pools(b, 2, 64, TYPES[ct], 4)
        cache, q = KVCache(kp, vp), rows((b.rows + 5, 4, 64), TYPES[rt], 5)
        plain, moved = b.device(new), b.device(new)
        moved = KVBatch(plain.q_start + 5, plain.pos0, plain.pages, rows=b.rows + 5, max_new=new)
        out = torch.full_like(q, 7.0)
        cache.attend(moved, q, out=out)
        assert bool((out[:5] == 7.0).all()) and torch.equal(out[5:], cache.attend(plain, q[5:].contiguous()))
        got = cache.append(moved, q, q[:, :2], q[:, 2:], q_out=torch.full_like(q, 7.0))
        assert bool((got[:5] == 7.0).all())
        assert torch.equal(got[5:], cache.append(plain, q[5:].contiguous(), q[5:, :2], q[5:, 2:]))
        cache.check()


def test_attend_bad_tables_touch_nothing():
    """Page ids outside the pool and positions past the table: reported once, the other sequences' rows
    right, later calls unaffected."""
    from cachepotato_b200 import CpgError
    from cachepotato_b200.kv import KVBatch, KVCache
    for rt, ct in COMBOS:
        for new in (1, 90):
            b = R.Batch([(1, 50), (new, 50), (1, 130)], 16, 6)
            kp, vp = R.pools(b, 2, 128, TYPES[ct], 7)
            q = rows((b.rows, 4, 128), TYPES[rt], 8)
            want, size = R.attend(b, q, kp, vp, 128 ** -0.5, 0)
            tol = attend_tol(b, want, size, vp, TYPES[rt])
            cache = KVCache(kp, vp, rope_dim=0)
            bad = b.device(new)
            ws = cache.workspace(4)
            good = bad.pages.clone()
            for wrong in (-5, b.n_pages, 2 ** 31 - 1):
                bad.pages[1, 2] = wrong
                got = cache.attend(bad, q, ws=ws)
                with pytest.raises(CpgError):
                    cache.check()
                cache.check()
                for s in (slice(0, 1), slice(1 + new, None)):
                    close(got[s], want[s], tol[s], "other rows")
                k, v = rows((b.rows, 2, 128), TYPES[rt], 9), rows((b.rows, 2, 128), TYPES[rt], 10)
                kp2 = kp.clone()
                keep = KVCache(kp2, vp.clone(), rope_dim=0)
                bad.pages[1, (50 + new - 1) // 16] = wrong
                keep.append(bad, q, k, v)
                with pytest.raises(CpgError):
                    keep.check()
                bad.pages.copy_(good)
            bad.pos0[1] = 2 ** 31 - 40                            # far past the table
            got = cache.attend(bad, q, ws=ws)
            with pytest.raises(CpgError):
                cache.check()
            close(got[:1], want[:1], tol[:1], "other rows")
            bad.pos0[1] = -3
            cache.attend(bad, q, ws=ws)
            with pytest.raises(CpgError):
                cache.check()
            bad.pos0[1] = 50
            close(cache.attend(bad, q, ws=ws), want, tol, "after")
            cache.check()


def bad_starts(good, T):
    """Starts no batch has, each with what is wrong about it."""
    lo, hi = -2 ** 31, 2 ** 31 - 1
    made = []
    for at, values in ((0, (lo, -1, hi)), (1, (lo, -7, hi, T + 1)), (2, (lo, 0, hi, T + 9)), (3, (lo, 0, 1, hi, T + 1))):
        for v in values:
            s = good.copy()
            s[at] = v
            made.append(s)
    return made + [good[::-1].copy(), np.full_like(good, lo), np.full_like(good, hi), np.array([hi, lo, hi, lo], np.int32)]


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("new", [1, 90])
def test_bad_starts_are_reported_and_touch_nothing(rt, ct, new):
    """Negative, descending and too large starts: both operators report them, once, and write nothing
    outside the rows, or outside the pages of the table; the next call is right."""
    from cachepotato_b200 import CpgError
    from cachepotato_b200.kv import KVBatch, KVCache
    H, KV, hd, page, guard = 8, 2, 64, 16, 8
    b = R.Batch([(1, 50), (new, 50), (2, 130)], page, 6, spare=9)
    kp, vp = R.pools(b, KV, hd, TYPES[ct], 7)
    T = b.rows
    free = torch.ones(b.n_pages, dtype=torch.bool, device="cuda")
    free[torch.from_numpy(b.table[b.table >= 0]).long().cuda()] = False
    qkv = rows((T + 2 * guard, H + 2 * KV, hd), TYPES[rt], 8)
    q, k, v = (qkv[guard:guard + T, x] for x in (slice(0, H), slice(H, H + KV), slice(H + KV, None)))
    cache = KVCache(kp, vp)
    good = b.device(new)
    ws = cache.workspace(H)
    out = torch.full((T + 2 * guard, H, hd), 7.0, dtype=TYPES[rt], device="cuda")
    inner = out[guard:guard + T]
    want_q = cache.append(good, q, k, v).clone()
    want = cache.attend(good, want_q, ws=ws)
    kept = [p.clone() for p in (kp, vp)]
    cache.check()
    for s in bad_starts(b.start, T):
        bad = KVBatch(torch.from_numpy(s).cuda(), good.pos0, good.pages, rows=T, max_new=new)
        for call in (lambda: cache.append(bad, q, k, v, q_out=inner), lambda: cache.attend(bad, want_q, out=inner, ws=ws)):
            call()
            with pytest.raises(CpgError):
                cache.check()
            cache.check()
            assert bool((out[:guard] == 7.0).all()) and bool((out[guard + T:] == 7.0).all()), s
            assert all(torch.equal(p[free], x[free]) for p, x in zip((kp, vp), kept)), s
        for p, x in zip((kp, vp), kept):
            p.copy_(x)
        assert torch.equal(cache.append(good, q, k, v), want_q) and torch.equal(cache.attend(good, want_q, ws=ws), want), s
        assert all(torch.equal(p, x) for p, x in zip((kp, vp), kept))
        cache.check()


@pytest.mark.parametrize("new", [1, 60])
def test_a_sequence_without_rows_may_stand_anywhere(new):
    """A padded batch: the position and the pages of a sequence that brings no rows are not looked at."""
    from cachepotato_b200.kv import KVCache
    b = R.Batch([(0, 5), (new, 50), (0, 9), (1, 130), (0, 0)], 16, 6)
    kp, vp = R.pools(b, 2, 64, torch.bfloat16, 7)
    q, k = rows((b.rows, 8, 64), torch.bfloat16, 8), rows((b.rows, 2, 64), torch.bfloat16, 9)
    cache, batch = KVCache(kp, vp), b.device(new)
    made = cache.append(batch, q, k, k)
    want = cache.attend(batch, made)
    batch.pos0[torch.tensor([0, 2, 4], device="cuda")] = torch.tensor([-1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device="cuda")
    batch.pages[torch.tensor([0, 2, 4], device="cuda")] = -1
    assert torch.equal(cache.append(batch, q, k, k), made) and torch.equal(cache.attend(batch, made), want)
    cache.check()


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("n", [3, 160, 170, 384, 400])
@pytest.mark.parametrize("chunk", [1, 40])
def test_every_bad_sequence_is_reported(rt, ct, n, chunk):
    """More sequences than a block has threads: the last one past its table, and all of them."""
    from cachepotato_b200 import CpgError
    from cachepotato_b200.kv import KVCache
    b = R.Batch([(chunk, 9)] + [(1, 5)] * (n - 1), 8, 6, wide=0)
    kp, vp = R.pools(b, 2, 64, TYPES[ct], 7)
    q, k = rows((b.rows, 8, 64), TYPES[rt], 8), rows((b.rows, 2, 64), TYPES[rt], 9)
    cache, batch = KVCache(kp, vp, rope_dim=0), b.device(chunk)
    ws = cache.workspace(8)
    calls = [lambda: cache.append(batch, q, k, k), lambda: cache.attend(batch, q, ws=ws)]
    want = [call() for call in calls]
    cache.check()
    pos0 = batch.pos0.clone()
    wide = b.table.shape[1] * 8
    for places in (slice(n - 1, n), slice(0, n)):
        for bad in (wide, 2 ** 31 - 40, -3):                      # one past the table, far past, in front
            batch.pos0[places] = bad
            for call in calls:
                call()
                with pytest.raises(CpgError):
                    cache.check()
                cache.check()
            batch.pos0.copy_(pos0)
    assert all(torch.equal(call(), w) for call, w in zip(calls, want))
    cache.check()


def test_empty_batches():
    from cachepotato_b200.kv import KVCache
    b = R.Batch([(0, 5), (0, 0)], 16, 1, pad=4)
    kp, vp = R.pools(b, 1, 64, torch.float32, 2)
    cache, q = KVCache(kp, vp), rows((4, 2, 64), torch.float32, 3)
    out = torch.full_like(q, 7.0)
    cache.attend(b.device(), q, out=out)
    cache.append(b.device(), q, q[:, :1], q[:, :1], q_out=out)
    cache.check()
    assert bool((out == 7.0).all())
    b = R.Batch([(0, 5)], 16, 1)
    none = torch.empty(0, 2, 64, device="cuda")
    assert cache.attend(b.device(), none).shape == (0, 2, 64)
    cache.append(b.device(), none, none[:, :1], none[:, :1])


@pytest.mark.parametrize("rt,ct", [("f32", "f32"), ("bf16", "bf16")])
def test_a_captured_step_follows_the_tables(rt, ct):
    """Append and attend captured once, replayed as the sequences grow; two graphs share the workspace
    and calls of other shapes run between the replays."""
    from cachepotato_b200.kv import KVBatch, KVCache
    H, KV, hd, page, n = 8, 2, 128, 16, 3
    g = torch.Generator().manual_seed(1)
    kp, vp = (torch.zeros(40, page, KV, hd, dtype=TYPES[ct], device="cuda") for _ in range(2))
    table = torch.randperm(40, generator=g)[:36].reshape(n, 12).to(torch.int32).cuda()
    pos0 = torch.tensor([0, 30, 100], dtype=torch.int32, device="cuda")
    start = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    cache = KVCache(kp, vp)
    ws = cache.workspace(H)
    batch = KVBatch(start, pos0, table, rows=n, max_new=1)
    other = R.Batch([(70, 20)], page, 2)
    other.n_pages = 40
    oq = rows((70, H, hd), TYPES[rt], 3)
    graphs, ins, outs = [], [], []
    stream = torch.cuda.Stream()
    for _ in range(2):
        qkv = torch.zeros(n, H + 2 * KV, hd, dtype=TYPES[rt], device="cuda")
        q2, out = torch.zeros(n, H, hd, dtype=TYPES[rt], device="cuda"), torch.zeros(n, H, hd, dtype=TYPES[rt], device="cuda")
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=stream):
            cache.append(batch, qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:], q_out=q2)
            cache.attend(batch, q2, out=out, ws=ws)
        graphs.append(gr); ins.append((qkv, q2)); outs.append(out)
    for step in range(24):
        which = step % 2
        ins[which][0].copy_(rows((n, H + 2 * KV, hd), TYPES[rt], 100 + step))
        graphs[which].replay()
        b = R.Batch([(1, int(c)) for c in pos0.tolist()], page, 0)
        b.table = table.cpu().numpy()
        want, size = R.attend(b, ins[which][1], kp, vp, hd ** -0.5, 0)
        close(outs[which], want, attend_tol(b, want, size, vp, TYPES[rt]), f"step {step}")
        cache.attend(other.device(70), oq, ws=ws)
        pos0 += 1
    cache.check()


def test_two_streams_and_another_stream():
    from cachepotato_b200.kv import KVCache
    b = R.Batch([(1, 3000), (1, 900)], 16, 3)
    kp, vp = R.pools(b, 2, 128, torch.bfloat16, 4)
    cache = KVCache(kp, vp, rope_dim=0)
    qs = [rows((2, 8, 128), torch.bfloat16, 5 + i) for i in range(2)]
    want = [cache.attend(b.device(1), q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    wss = [cache.workspace(8) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [cache.attend(b.device(1), q, ws=w, stream=s) for q, w, s in zip(qs, wss, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_outputs_made_for_another_stream():
    """What the calls allocate is free on the stream that writes it: not a block that the current stream
    has given back but is still using."""
    from cachepotato_b200.kv import KVCache
    b = R.Batch([(40, 30), (1, 5)], 16, 3)
    kp, vp = R.pools(b, 2, 64, torch.float32, 4)
    cache, batch = KVCache(kp, vp), b.device(40)
    q, k = rows((b.rows, 8, 64), torch.float32, 5), rows((b.rows, 2, 64), torch.float32, 6)
    ws = cache.workspace(8)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    given_back = []
    for _ in range(4):                                            # blocks of the outputs' size, freed on the current stream
        given_back.append(torch.empty_like(q))
    places = {t.data_ptr() for t in given_back}
    del given_back
    made = cache.append(batch, q, k, k, stream=side)
    out = cache.attend(batch, made, ws=ws, stream=side)
    assert made.data_ptr() not in places and out.data_ptr() not in places
    side.synchronize()
    want = cache.attend(batch, cache.append(batch, q, k, k), ws=ws)
    assert torch.equal(out, want)
    with pytest.raises(CpgError):
        cache.append(batch, None, k, k, q_out=q)


def test_a_new_cache_on_another_stream():
    """A stream that does not wait for the default one sees a handle's angles as soon as there is a handle."""
    from cachepotato_b200.kv import KVCache
    b = R.Batch([(40, 300), (1, 5)], 16, 3)
    kp, vp = R.pools(b, 2, 64, torch.float32, 4)
    batch = b.device(40)
    q, k = rows((b.rows, 8, 64), torch.float32, 5), rows((b.rows, 2, 64), torch.float32, 6)
    made = torch.empty_like(q)
    side = torch.cuda.Stream()
    for theta in (1e4, 5e5, 1e6, 77.0):
        torch.cuda.synchronize()
        cache = KVCache(kp, vp, rope_theta=theta)
        cache.append(batch, q, k, k, q_out=made, stream=side)
        side.synchronize()
        assert torch.equal(made, cache.append(batch, q, k, k))
        cache.check()


def test_windows_past_every_position():
    """Windows are whole numbers of any size: one that no int holds is not cut to its low bits."""
    from cachepotato_b200 import CpgError
    from cachepotato_b200.kv import KVCache
    for rt, ct in COMBOS:
        for new in (1, 90):
            b = R.Batch([(new, 500), (new, 3)], 16, 8)
            kp, vp = R.pools(b, 1, 64, TYPES[ct], 9)
            q = rows((b.rows, 8, 64), TYPES[rt], 10)
            cache, batch = KVCache(kp, vp, rope_dim=0), b.device(new)
            want = cache.attend(batch, q)
            for window in (500 + new, 2 ** 31 - 1, 2 ** 31 + 7, 2 ** 32 + 5, 2 ** 63):
                assert torch.equal(cache.attend(batch, q, window=window), want), window
            for window in (-1, -2 ** 31, 5 - 2 ** 32):
                with pytest.raises(CpgError):
                    cache.attend(batch, q, window=window)


@pytest.mark.parametrize("rt,ct", COMBOS)
def test_windows_as_long_as_the_table(rt, ct):
    """Windows on both sides of what the table holds give the same rows as none."""
    from cachepotato_b200.kv import KVCache
    for new in (1, 90):
        b = R.Batch([(new, 500), (new, 3)], 16, 8)
        kp, vp = R.pools(b, 2, 64, TYPES[ct], 9)
        poison(b, kp, vp)
        q = rows((b.rows, 8, 64), TYPES[rt], 10)
        cache, batch = KVCache(kp, vp, rope_dim=0), b.device(new)
        want, held = cache.attend(batch, q), b.table.shape[1] * 16
        for window in (500 + new, held - 1, held, held + 1, 2 ** 31 - 1):
            assert torch.equal(cache.attend(batch, q, window=window), want), window
        cache.check()


def test_scales_too_large_are_refused():
    """Past 2.3e38 the scale in powers of two leaves f32: such a call would give nothing but NaN."""
    from cachepotato_b200 import CpgError
    from cachepotato_b200.kv import KVCache
    b = R.Batch([(2, 50)], 16, 8)
    kp, vp = R.pools(b, 1, 64, torch.bfloat16, 9)
    q = rows((b.rows, 8, 64), torch.bfloat16, 10)
    cache, batch = KVCache(kp, vp, rope_dim=0), b.device(2)
    for scale in (3e38, 2.4e38):
        with pytest.raises(CpgError):
            cache.attend(batch, q, scale=scale)


def test_attend_is_the_same_every_time():
    """Work split over blocks is joined in a fixed order."""
    from cachepotato_b200.kv import KVCache
    for rt, ct in COMBOS:
        for lens in ([(1, 9000), (1, 77)], [(300, 700), (1, 2000)]):
            b = R.Batch(lens, 16, 3)
            kp, vp = R.pools(b, 2, 128, TYPES[ct], 4)
            cache, q = KVCache(kp, vp, rope_dim=0), rows((b.rows, 8, 128), TYPES[rt], 5)
            ws, batch = cache.workspace(8), b.device(max(n for n, _ in lens))
            first = cache.attend(batch, q, ws=ws)
            for _ in range(5):
                assert torch.equal(cache.attend(batch, q, ws=ws), first)


@pytest.mark.parametrize("rt,ct", COMBOS)
@pytest.mark.parametrize("window", [0, 200])
def test_attend_when_tiles_come_late(rt, ct, window):
    """Pages out of memory instead of the L2 cache: tiles of keys and values arrive late and in no order,
    and every stage of the kernels waits for every other at some time. The same bits each time."""
    from cachepotato_b200.kv import KVCache
    lens = [(100 + 9 * i, 37 * i) for i in range(24)] + [(1, 900), (520, 0)]
    b = R.Batch(lens, 16, 12)
    kp, vp = R.pools(b, 2, 128, TYPES[ct], 13)
    poison(b, kp, vp)
    q = rows((b.rows, 16, 128), TYPES[rt], 14)
    want, size = R.attend(b, q, kp, vp, 128 ** -0.5, window)
    cache, batch = KVCache(kp, vp, rope_dim=0), b.device(520)
    other = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    first = None
    for i in range(20):
        other.fill_(i)                                            # more than L2 holds
        got = cache.attend(batch, q, window=window)
        first = got.clone() if first is None else first
        assert torch.equal(got, first), i
    close(first, want, attend_tol(b, want, size, vp, TYPES[rt]), "late tiles")
    cache.check()


def test_long_cache_offsets_past_32_bits():
    """A pool of more than 2^32 elements: the last pages are reached."""
    from cachepotato_b200.kv import KVCache
    page, KV, hd = 256, 8, 128
    n_pages = (2 ** 32) // (page * KV * hd) + 9                   # 8.6 GB a pool at 16 bits
    kp, vp = (torch.zeros(n_pages, page, KV, hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for new in (1, 40):
        b = R.Batch([(new, 600)], page, 1)
        b.table[0, :3] = [n_pages - 1, n_pages - 5, n_pages - 2]
        q, k, v = (rows((new, h, hd), torch.bfloat16, 2 + h) for h in (16, 8, 8))
        cache = KVCache(kp, vp)
        for p, s in ((kp, 5), (vp, 6)):
            p[n_pages - 5:] = rows((5, page, KV, hd), torch.bfloat16, s)
        low = R.Batch([(new, 600)], page, 1)
        low.n_pages, low.table[0, :3] = 5, [4, 0, 3]
        lk, lv = kp[n_pages - 5:].clone(), vp[n_pages - 5:].clone()
        small = KVCache(lk, lv)
        got = cache.attend(b.device(new), cache.append(b.device(new), q, k, v))
        want = small.attend(low.device(new), small.append(low.device(new), q, k, v))
        cache.check()
        assert torch.equal(got, want) and torch.equal(kp[n_pages - 5:], lk) and torch.equal(vp[n_pages - 5:], lv)
        assert not kp[:n_pages - 5].any()


# ---------------------------------------------------------------------------------------- refusals
def test_refusals():
    from cachepotato_b200 import CpgError
    from cachepotato_b200.kv import KVBatch, KVCache
    z = lambda *s, dt=torch.bfloat16: torch.zeros(s, dtype=dt, device="cuda")
    b = R.Batch([(2, 30)], 16, 1)
    kp, vp = R.pools(b, 2, 128, torch.bfloat16, 2)
    cache, batch = KVCache(kp, vp), b.device()
    q, k = z(2, 4, 128), z(2, 2, 128)
    bad_pools = [(kp, vp.float()), (kp, vp[:-1]), (kp.cpu(), vp.cpu()), (kp.to(torch.float64), vp.to(torch.float64)),
                 (kp[..., :96], vp[..., :96]), (kp[:, :12], vp[:, :12]), (kp.transpose(2, 3), vp.transpose(2, 3)),
                 (kp[0], vp[0]), (kp, vp.transpose(1, 2).contiguous().transpose(1, 2))]
    for p in bad_pools:
        with pytest.raises(CpgError):
            KVCache(*p)
    for kw in (dict(rope_dim=8), dict(rope_dim=144), dict(rope_theta=0.0), dict(rope_theta=float("nan"))):
        with pytest.raises(CpgError):
            KVCache(kp, vp, **kw)
    wrong = [lambda: cache.attend(batch, z(2, 3, 128)), lambda: cache.attend(batch, z(3, 4, 128)),
             lambda: cache.attend(batch, z(2, 4, 64)), lambda: cache.attend(batch, z(2, 4, 128, dt=torch.float16)),
             lambda: cache.attend(batch, q, scale=0.0), lambda: cache.attend(batch, q, scale=float("inf")),
             lambda: cache.attend(batch, q, window=-1), lambda: cache.attend(batch, q, out=z(2, 4, 128, dt=torch.float32)),
             lambda: cache.attend(batch, z(2, 128, 4).transpose(1, 2)), lambda: cache.attend(batch, z(2, 4, 132)[..., 4:]),
             lambda: cache.attend(batch, q, ws=z(64, dt=torch.uint8)), lambda: cache.attend(batch, q.cpu()),
             lambda: cache.append(batch, q, k, z(2, 3, 128)), lambda: cache.append(batch, q.float(), k, k),
             lambda: cache.append(batch, q, k.half(), k.half()), lambda: cache.append(batch, q, k, k, q_norm=z(128)),
             lambda: cache.append(batch, q, k, k, k_norm=z(64, dt=torch.float32)),
             lambda: cache.append(batch, q, k, k, eps=-1.0), lambda: cache.append(batch, q, k, k, eps=float("nan"))]
    for call in wrong:
        with pytest.raises(CpgError):
            call()
    i32 = dict(dtype=torch.int32, device="cuda")
    s, p0, tab = torch.zeros(3, **i32), torch.zeros(2, **i32), torch.zeros(2, 4, **i32)
    for args, rows_ in (((s[:2], p0, tab), 1), ((s, p0, tab[:1]), 1), ((s.long(), p0, tab), 1), ((s, p0.cpu(), tab), 1),
                        ((s, p0, tab[0]), 1), ((s, p0, tab), -1), ((s, p0, torch.zeros(4, 2, **i32).t()), 1)):
        with pytest.raises(CpgError):
            KVBatch(*args, rows=rows_)


def test_c_entry_refusals():
    from cachepotato_b200 import _lib
    L = _lib.lib()
    pool = torch.zeros(1 << 16, dtype=torch.float32, device="cuda")
    p = pool.data_ptr()

    def create(**kw):
        d = dict(n_kv=2, head_dim=64, page_size=16, n_pages=4, type=0, k=p, v=p, page_stride=2048, pos_stride=128,
                 head_stride=64, rope_dim=64, rope_theta=1e4, rope_f32=0)
        d.update(kw)
        h = ctypes.c_void_p()
        rc = L.cpg_kv_create(ctypes.byref(_lib.KvDesc(**d)), ctypes.byref(h))
        assert (rc == 0) == bool(h.value)
        return rc, h
    for kw in (dict(n_kv=0), dict(head_dim=96), dict(page_size=12), dict(page_size=0), dict(n_pages=0), dict(type=3), dict(k=None),
               dict(v=p + 4), dict(pos_stride=126), dict(head_stride=32), dict(page_stride=1024), dict(pos_stride=64),
               dict(rope_dim=24), dict(rope_dim=-16), dict(rope_theta=-1.0)):
        assert create(**kw)[0] == _lib.CPG_EINVAL, kw
    rc, h = create()
    assert rc == 0
    assert L.cpg_kv_attend_workspace_bytes(h, 3) == 0 and L.cpg_kv_attend_workspace_bytes(None, 2) == 0
    n = L.cpg_kv_attend_workspace_bytes(h, 2)
    ints = torch.zeros(8, dtype=torch.int32, device="cuda").data_ptr()
    ok = dict(n_seqs=1, rows=1, q_start=ints, pos0=ints, pages=ints, table_stride=1, max_pages=1, max_new=1)
    call = lambda b, **kw: L.cpg_kv_attend(h, ctypes.byref(_lib.KvRows(**{**ok, **b})), kw.get("type", 0), kw.get("heads", 2),
                                           kw.get("q", p), kw.get("stride", 128), kw.get("out", p), 128, 1.0, 0,
                                           kw.get("ws", p), kw.get("bytes", n), None)
    for b, kw in ((dict(n_seqs=-1), {}), (dict(rows=-1), {}), (dict(pages=None), {}), (dict(max_pages=0), {}),
                  (dict(table_stride=0), {}), ({}, dict(type=1)), ({}, dict(heads=3)), ({}, dict(heads=0)), ({}, dict(q=None)),
                  ({}, dict(q=p + 4)), ({}, dict(stride=64)), ({}, dict(stride=130)), ({}, dict(out=None)), ({}, dict(ws=None)),
                  ({}, dict(ws=p + 16)), ({}, dict(bytes=n - 1))):
        assert call(b, **kw) == _lib.CPG_EINVAL, (b, kw)
        assert _lib.last_error()
    assert L.cpg_kv_append(None, None, 0, 1, p, 64, p, 128, p, 128, None, None, 0.0, p, 64, None) == _lib.CPG_EINVAL
    assert L.cpg_kv_check(None, None) == _lib.CPG_EINVAL
    L.cpg_kv_destroy(h)
    L.cpg_kv_destroy(None)
