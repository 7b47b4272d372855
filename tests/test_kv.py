"""The paged cache's refusals that need no GPU: every argument is checked before the first CUDA call."""
import ctypes

import pytest

from cachepotato_b200 import CpgError, _lib


def _desc(**kw):
    d = dict(n_kv=2, head_dim=64, page_size=16, n_pages=4, type=0, k=1 << 20, v=1 << 21, page_stride=2048, pos_stride=128,
             head_stride=64, rope_dim=64, rope_theta=1e4, rope_f32=0)
    d.update(kw)
    return _lib.KvDesc(**d)


BAD = [dict(n_kv=0), dict(n_kv=2000), dict(head_dim=96), dict(head_dim=0), dict(page_size=12), dict(page_size=0), dict(page_size=-8),
       dict(page_size=1 << 17), dict(n_pages=0), dict(n_pages=-1), dict(type=3), dict(type=-1), dict(k=None), dict(v=None),
       dict(v=(1 << 21) + 4), dict(pos_stride=126), dict(pos_stride=130), dict(head_stride=32), dict(head_stride=-64),
       dict(page_stride=1024), dict(pos_stride=64), dict(page_stride=1 << 40), dict(rope_dim=24), dict(rope_dim=-16),
       dict(rope_dim=80), dict(rope_theta=0.0), dict(rope_theta=-1.0), dict(rope_theta=float("nan")), dict(rope_theta=float("inf"))]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_create_refuses(kw):
    L = _lib.lib()
    h = ctypes.c_void_p(1)
    assert L.cpg_kv_create(ctypes.byref(_desc(**kw)), ctypes.byref(h)) == _lib.CPG_EINVAL
    assert h.value is None and "cpg_kv_create" in _lib.last_error()


def test_null_handles_are_refused():
    L = _lib.lib()
    h = ctypes.c_void_p()
    assert L.cpg_kv_create(None, ctypes.byref(h)) == _lib.CPG_EINVAL
    assert L.cpg_kv_create(ctypes.byref(_desc()), None) == _lib.CPG_EINVAL
    rows = ctypes.byref(_lib.KvRows(1, 1, 16, 16, 16, 1, 1, 1))
    assert L.cpg_kv_append(None, rows, 0, 2, 16, 128, 16, 128, 16, 128, None, None, 0.0, 16, 128, None) == _lib.CPG_EINVAL
    assert L.cpg_kv_attend(None, rows, 0, 2, 16, 128, 16, 128, 1.0, 0, 256, 1 << 30, None) == _lib.CPG_EINVAL
    assert L.cpg_kv_check(None, None) == _lib.CPG_EINVAL
    assert L.cpg_kv_attend_workspace_bytes(None, 2) == 0
    L.cpg_kv_destroy(None)
    p = ctypes.c_void_p(1)
    assert L.cpg_qwen3_paged_create(None, 1, 8, 8, 1, 0, ctypes.byref(p)) == _lib.CPG_EINVAL
    assert L.cpg_qwen3_paged_step(None, None, None, None, 1, None) == _lib.CPG_EINVAL
    assert L.cpg_qwen3_paged_generate(None, None, None, 1, 1, None) == _lib.CPG_EINVAL
    assert L.cpg_qwen3_paged_drop(None, 0) == _lib.CPG_EINVAL
    assert L.cpg_qwen3_paged_position(None, 0) == -1 and L.cpg_qwen3_paged_free_pages(None) == 0
    L.cpg_qwen3_paged_destroy(None)


def test_host_tensors_are_refused():
    torch = pytest.importorskip("torch")
    from cachepotato_b200.kv import KVBatch, KVCache
    pool = torch.zeros(4, 16, 2, 64)
    with pytest.raises(CpgError):
        KVCache(pool, pool)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(CpgError):
        KVBatch(i, i[:1], i.view(1, 2), rows=1)
