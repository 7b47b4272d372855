"""Many sequences over a pool of pages (cpg_qwen3_paged).

Oracle: the model's own greedy path (cpg_qwen3_generate, which tests/test_gpu_qwen3.py holds to the
reference engine's cp_chat loop) on each sequence alone: with an f32 cache every slot must produce
exactly its ids however prompts are cut into chunks and steps are mixed."""
import numpy as np
import pytest

import oracle as O
from conftest import max_rel
from helpers import BLOCK_TOL, device_model

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def _small(orc, seed):
    return O.SynthModel(256, 4, 2, 128, 256, 16, 4, 512, 2, seed=seed, norm_jitter=0.1, oracle=orc)


def _prompts(vocab, lens, seed):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, vocab, n).astype(np.int32) for n in lens]


@pytest.mark.parametrize("page,chunk", [(8, 100), (16, 7), (64, 1)])
def test_mixed_steps_match_each_sequence_alone(orc, page, chunk):
    """Sequences join at different steps, their prompts read `chunk` tokens a step while the others
    generate; one leaves and its pages are reused."""
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 61)
    prompts = _prompts(m.vocab, [19, 3, 41, 1, 12], 62)
    n_new = 6
    gm = device_model(m, max_ctx=128)
    p = Qwen3Paged(gm, 3, 64, n_pages=3 * 64 // page, page_size=page)
    total = p.free_pages()
    got = {i: [] for i in range(len(prompts))}
    fed = {i: 0 for i in got}
    waiting, running = list(got), {}                              # running: slot -> sequence
    logits = {}
    try:
        steps = 0
        while waiting or running:
            if waiting and steps % 2 == 0 and len(running) < 3:   # a new sequence every other step
                slot = next(s for s in range(3) if s not in running)
                running[slot] = waiting.pop(0)
            slots, chunks = [], []
            for slot, i in sorted(running.items(), reverse=steps % 2):
                rest = prompts[i][fed[i]:fed[i] + chunk]
                slots.append(slot)
                chunks.append(rest if len(rest) else [got[i][-1]])
            out = p.step(slots, chunks)
            lg = p.logits().cpu().numpy()
            for r, (slot, c) in enumerate(zip(slots, chunks)):
                i = running[slot]
                fed[i] += len(c)
                assert p.position(slot) == fed[i]
                if fed[i] >= len(prompts[i]):
                    got[i].append(int(out[r]))
                    logits[i] = lg[r]
                if len(got[i]) == n_new + 1:
                    p.drop(slot)
                    assert p.position(slot) == -1
                    del running[slot]
            steps += 1
        assert p.free_pages() == total
        for i, prompt in enumerate(prompts):
            assert got[i] == gm.generate(prompt, n_new).tolist(), i
            assert max_rel(logits[i], gm.logits().cpu().numpy()) <= BLOCK_TOL
    finally:
        p.close()
        gm.close()


@pytest.mark.parametrize("n", [1, 4, 12])
def test_generate_matches_each_sequence_alone(orc, n):
    """Captured steps of n sequences; 12 run their projections and head on the dense kernel."""
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 71)
    prompts = _prompts(m.vocab, list(range(1, n + 1)), 72)
    gm = device_model(m, max_ctx=96)
    p = Qwen3Paged(gm, n, 40, n_pages=5 * n, page_size=8)
    try:
        first = p.step(np.arange(n), prompts)
        order = np.arange(n)[::-1].copy()
        a = p.generate(order, first[order], 4)
        b = p.generate(order, a[-1], 3)
        for r, j in enumerate(order):
            want = gm.generate(prompts[j], 7)
            assert [int(first[j])] + a[:, r].tolist() + b[:, r].tolist() == want.tolist(), j
            assert p.position(j) == len(prompts[j]) + 7
    finally:
        p.close()
        gm.close()


@pytest.mark.parametrize("cache,tol", [("f32", BLOCK_TOL), ("f16", 16 * 2.0 ** -11), ("bf16", 16 * 2.0 ** -8)])
def test_cache_types(orc, cache, tol):
    """Logits after a chunked prompt and a few tokens against the model's own path. 16-bit caches round
    each key and value by half a step; scores of size up to 8 carry that eight times over into the
    weights, and two layers add theirs: 16 half steps."""
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 81)
    prompt = _prompts(m.vocab, [50], 82)[0]
    gm = device_model(m, max_ctx=96)
    p = Qwen3Paged(gm, 2, 96, n_pages=12, page_size=16, cache=cache)
    try:
        gm.prefill(prompt)
        want = gm.logits().cpu().numpy()
        p.step([1], [prompt[:33]])
        p.step([1, 0], [prompt[33:], prompt[:5]])
        assert max_rel(p.logits()[0].cpu().numpy(), want) <= tol
        gm.prefill(prompt[:5])
        assert max_rel(p.logits()[1].cpu().numpy(), gm.logits().cpu().numpy()) <= tol
    finally:
        p.close()
        gm.close()


def test_paged_leaves_the_models_own_sequence_alone(orc):
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 25)
    a, b = _prompts(m.vocab, [6, 3], 26)
    gm = device_model(m, max_ctx=32)
    try:
        plain = gm.generate(a, 4).tolist()
        p = Qwen3Paged(gm, 2, 32, n_pages=4, page_size=16, cache="bf16")
        try:
            seq = [gm.prefill(a)]
            p.step([1], [b])
            for _ in range(4):
                seq.append(gm.step(seq[-1]))
                p.step([1], [[seq[-1] % m.vocab]])
        finally:
            p.close()
    finally:
        gm.close()
    assert seq == plain


def test_qwen3_widths(orc):
    """Qwen3-30B-A3B widths: a chunk of 40 beside 20 single tokens, projections on tcgen05."""
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = O.SynthModel(2048, 32, 4, 128, 768, 128, 8, 4096, 2, seed=27, norm_jitter=0.05, oracle=orc)
    prompts = _prompts(m.vocab, np.random.default_rng(28).integers(1, 7, 20), 29)
    long = _prompts(m.vocab, [48], 30)[0]
    gm = device_model(m, max_ctx=128)
    p = Qwen3Paged(gm, 21, 64, n_pages=100, page_size=16)
    try:
        nxt = p.step(np.arange(20), prompts)
        got = [[int(x)] for x in nxt]
        p.step([20], [long[:8]])
        out = p.step(np.arange(21), [[x] for x in nxt] + [long[8:]])
        for j in range(20):
            got[j].append(int(out[j]))
        lg = p.logits().cpu().numpy()
        for j in range(20):
            assert got[j] == gm.generate(prompts[j], 1).tolist(), j
        gm.prefill(long)
        assert max_rel(lg[20], gm.logits().cpu().numpy()) <= BLOCK_TOL
    finally:
        p.close()
        gm.close()


def test_refusals_change_nothing(orc):
    from cachepotato_b200 import CpgError, _lib
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 31)
    gm = device_model(m, max_ctx=64)
    for kw in (dict(n_pages=0), dict(n_pages=4, page_size=12), dict(n_pages=4, page_size=0), dict(n_pages=4, cache="fp8")):
        with pytest.raises(CpgError):
            Qwen3Paged(gm, 3, 32, **kw)
    for args in ((0, 32), (65, 32), (3, 0)):
        with pytest.raises(CpgError):
            Qwen3Paged(gm, *args, n_pages=4)
    p = Qwen3Paged(gm, 3, 32, n_pages=4, page_size=8)
    try:
        n0 = int(p.step([0], [[1, 2, 3]])[0])
        free = p.free_pages()
        assert free == 3
        for slots, chunks in (([0, 0], [[1], [2]]), ([3], [[1]]), ([-1], [[1]]), ([0], [[m.vocab]]), ([0], [[]]),
                              ([0], [[-1]]), ([0], [np.arange(30)]), ([1], [np.zeros(65)]), ([], [])):
            with pytest.raises(CpgError):
                p.step(slots, chunks)
        with pytest.raises(CpgError) as e:                        # 4 pages asked for, 3 free
            p.step([1, 0], [np.ones(25, np.int32), [n0]])
        assert e.value.code == _lib.CPG_ENOMEM
        with pytest.raises(CpgError):
            p.generate([1], [1], 2)                               # slot 1 holds no sequence
        with pytest.raises(CpgError):
            p.generate([0], [n0], 30)                             # 3 + 30 positions > 32
        with pytest.raises(CpgError):
            p.generate([0], [n0], 0)
        with pytest.raises(CpgError):
            p.drop(7)
        assert p.position(0) == 3 and p.position(1) == -1 and p.free_pages() == free
        want = gm.generate([1, 2, 3], 20).tolist()
        assert [n0] + p.generate([0], [n0], 20)[:, 0].tolist() == want
    finally:
        p.close()
        gm.close()


def test_pools_no_memory_holds(orc):
    """Sizes past 64 bits are refused before anything is allocated, ones past the device's memory by the
    allocation; the model goes on."""
    from cachepotato_b200 import CpgError, _lib
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 71)
    gm = device_model(m, max_ctx=64)
    try:
        for n_pages, page in ((2**31 - 1, 8), (2**31 - 1, 65536), (2000, 65536)):
            with pytest.raises(CpgError) as e:
                Qwen3Paged(gm, 2, 64, n_pages=n_pages, page_size=page)
            assert e.value.code == _lib.CPG_ENOMEM
        p = Qwen3Paged(gm, 2, 64, n_pages=8, page_size=16)
        ids = _prompts(m.vocab, [9], 72)[0]
        assert p.step([1], [ids])[0] == gm.generate(ids, 1)[0]
        p.close()
    finally:
        gm.close()


def _report(p, page, n_pages, max_ctx, bits):
    """Puts `bits` into the cache's status word, where a kernel whose wait gave up leaves them. (No call
    hands the word out: it is found through the handles, whose members in front of it are checked.)"""
    import ctypes
    from cachepotato_b200.workload import device_view
    at = lambda where, n, t: [x for x in (t * n).from_address(where)]
    h = p.handle.value
    assert at(h + 8, 5, ctypes.c_int) == [p.n_slots, max_ctx, page, -(-max_ctx // page), n_pages]
    kv = at(at(h + 40, 1, ctypes.c_void_p)[0], 1, ctypes.c_void_p)[0]       # the vector's first handle
    assert at(kv + 40, 2, ctypes.c_int) == [page, n_pages]
    word = device_view(torch, at(kv + 56, 1, ctypes.c_void_p)[0], 4, "i4")
    assert int(word[0]) == 0
    word.fill_(bits)
    torch.cuda.synchronize()


def test_a_step_that_failed_can_be_repeated(orc):
    """A step whose kernels report that a wait gave up moves no position: the same call again writes the
    same places, and the ids are the model's."""
    from cachepotato_b200 import CpgError, _lib
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 91)
    a, b = _prompts(m.vocab, [11, 5], 92)
    gm = device_model(m, max_ctx=64)
    p = Qwen3Paged(gm, 2, 64, n_pages=16, page_size=8)
    timeout = 4

    def twice(call, before):
        rows = tuple(p.logits().shape) if before != (-1, -1) else None
        _report(p, 8, 16, 64, timeout)
        with pytest.raises(CpgError) as e:
            call()
        assert e.value.code == _lib.CPG_ETIMEOUT
        assert (p.position(0), p.position(1)) == before
        assert rows is None or tuple(p.logits().shape) == rows
        return call()
    try:
        x = twice(lambda: p.step([1, 0], [a[:7], b]), (-1, -1))
        x = twice(lambda: p.step([1], [a[7:]]), (5, 7)).tolist() + x[1:].tolist()        # slots 1, 0
        y = twice(lambda: p.step([1, 0], [[i] for i in x]), (5, 11)).tolist()
        z = twice(lambda: p.generate([0, 1], [y[1], y[0]], 3), (6, 12))
        assert (p.position(0), p.position(1)) == (9, 15) and p.free_pages() == 16 - 2 - 2
        for prompt, got in ((a, [x[0], y[0]] + z[:, 1].tolist()), (b, [x[1], y[1]] + z[:, 0].tolist())):
            assert got == gm.generate(prompt, 4).tolist()
    finally:
        p.close()
        gm.close()


def test_tables_are_no_wider_than_the_pool(orc):
    """max_ctx bounds positions, not memory: 64 tables of a billion positions over eight pages."""
    from cachepotato_b200 import CpgError, _lib
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 93)
    ids = _prompts(m.vocab, [60], 94)[0]
    gm = device_model(m, max_ctx=64)
    free = torch.cuda.mem_get_info()[0]
    p = Qwen3Paged(gm, 64, 1 << 30, n_pages=8, page_size=8)
    try:
        assert free - torch.cuda.mem_get_info()[0] < 1 << 29
        first = p.step([63], [ids])
        assert [int(first[0])] + p.generate([63], first, 4)[:, 0].tolist() == gm.generate(ids, 4).tolist()
        with pytest.raises(CpgError) as e:
            p.step([63], [[1]])
        assert e.value.code == _lib.CPG_ENOMEM and p.position(63) == 64 and p.free_pages() == 0
    finally:
        p.close()
        gm.close()


def test_the_model_may_be_closed_first(orc):
    """A pool left over by its model can still be closed, and closed twice."""
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 95)
    for _ in range(3):
        gm = device_model(m, max_ctx=64)
        p = Qwen3Paged(gm, 2, 64, n_pages=8, page_size=16)
        p.step([0], [[1, 2, 3]])
        gm.close()
        p.close()
        p.close()


def test_more_sequences_than_the_dense_kernels_take(orc):
    """72 slots: projections and head on the paths for larger steps, prompts and single tokens."""
    from cachepotato_b200.qwen3 import Qwen3Paged
    n = 72
    m = _small(orc, 97)
    prompts = _prompts(m.vocab, [1 + j % 4 for j in range(n)], 98)
    gm = device_model(m, max_ctx=256)
    p = Qwen3Paged(gm, n, 16, n_pages=2 * n, page_size=8)
    try:
        first = p.step(np.arange(n), prompts)
        assert tuple(p.logits().shape) == (n, m.vocab)
        order = np.random.default_rng(99).permutation(n).astype(np.int32)
        out = p.generate(order, first[order], 5)
        for r, j in enumerate(order):
            assert [int(first[j])] + out[:, r].tolist() == gm.generate(prompts[j], 5).tolist(), j
    finally:
        p.close()
        gm.close()


def test_a_chunk_is_one_row_of_ids(orc):
    """A table of ids is refused, not cut to the length of its first axis."""
    from cachepotato_b200 import CpgError
    from cachepotato_b200.qwen3 import Qwen3Paged
    m = _small(orc, 101)
    ids = _prompts(m.vocab, [6], 102)[0]
    gm = device_model(m, max_ctx=64)
    p = Qwen3Paged(gm, 2, 32, n_pages=4, page_size=16)
    try:
        for chunk in (ids[None], ids[:, None], ids.reshape(2, 3)):
            with pytest.raises(CpgError):
                p.step([0], [chunk])
        assert p.position(0) == -1 and p.free_pages() == 4
        assert p.step([0], ids[None])[0] == gm.generate(ids, 1)[0]        # (one chunk: the table's row)
    finally:
        p.close()
        gm.close()
