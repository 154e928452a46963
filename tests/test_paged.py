"""Refusals of the paged serving operators: arguments that the entry points turn
into errors before any device work (no GPU needed), and the Python checks."""
import ctypes
import os

import pytest

from torchless_b200 import LIB_PATH, lib, tl_paged_cache

pytestmark = pytest.mark.skipif(not os.path.exists(LIB_PATH), reason="library not built")
INVALID, UNSUPPORTED = 1, 2
A = 1 << 12  # a 16-byte aligned address that nothing reads


def cache(**kw):
    f = dict(k=A, v=A, n_blocks=8, n_kv_heads=2, block_size=16, head_dim=64, block_stride=2 * 16 * 64, dtype=1)
    f.update(kw)
    return tl_paged_cache(**f)


BAD_CACHES = [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(dtype=3), INVALID), (dict(head_dim=96), UNSUPPORTED),
    (dict(head_dim=0), UNSUPPORTED), (dict(block_size=12), UNSUPPORTED), (dict(block_size=4), UNSUPPORTED),
    (dict(block_size=512), UNSUPPORTED), (dict(n_blocks=0), INVALID), (dict(n_blocks=1 << 28), INVALID),
    (dict(n_kv_heads=0), INVALID), (dict(block_stride=2 * 16 * 64 - 8), INVALID),
    (dict(block_stride=2 * 16 * 64 + 1), INVALID), (dict(k=A + 8), INVALID),
]


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_bad_caches_are_refused(kw, status):
    L, c = lib(), ctypes.byref(cache(**kw))
    n = ctypes.c_size_t()
    assert L.tl_paged_attention_workspace(c, 1, 4, 1, 1, ctypes.byref(n)) == status
    assert L.tl_paged_attention(A, A, 256, c, A, 1, A, A, 1, 1, 4, 1.0, 0, A, 1 << 20, None) == status
    assert L.tl_qk_norm_rope(A, c, A, 0, 512, A, A, A, A, 9, 64, None, None, 1e-5, 1, 4, None) == status
    assert L.tl_last_error()


def test_attention_refusals():
    L, c = lib(), cache()

    def call(out=A, q=A, stride=256, table=A, width=1, start=A, lens=A, n_seq=1, n=1, heads=4, scale=1.0, ws=A,
             size=1 << 30):
        return L.tl_paged_attention(out, q, stride, ctypes.byref(c), table, width, start, lens, n_seq, n, heads, scale,
                                    0, ws, size, None)

    for kw in (dict(out=None), dict(q=None), dict(table=None), dict(start=None), dict(lens=None), dict(heads=3),
               dict(heads=0), dict(stride=248), dict(stride=257), dict(out=A + 4), dict(q=A + 2), dict(width=0),
               dict(width=1 << 31), dict(n=1 << 30), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert call(**kw) == INVALID, kw
    # nothing to do is not an error
    assert call(n=0, q=None, out=None) == 0
    assert call(n_seq=0) == 0


def test_scales_that_pass_fp32_are_refused():
    L, c = lib(), cache()
    for scale in (3.0e38, -3.0e38):
        assert L.tl_paged_attention(A, A, 256, ctypes.byref(c), A, 1, A, A, 1, 1, 4, scale, 0, A, 1 << 30, None) == INVALID


def test_rope_refusals():
    L, c = lib(), cache()

    def call(out=A, qkv=A, dtype=0, stride=512, pos=A, slots=A, cos=A, sin=A, n_pos=9, rot=64, wq=None, wk=None, n=1,
             heads=4):
        return L.tl_qk_norm_rope(out, ctypes.byref(c), qkv, dtype, stride, pos, slots, cos, sin, n_pos, rot, wq, wk,
                                 1e-5, n, heads, None)

    for kw in (dict(out=None), dict(qkv=None), dict(pos=None), dict(slots=None), dict(cos=None), dict(sin=None),
               dict(dtype=7), dict(stride=508), dict(stride=513), dict(n_pos=0), dict(heads=0), dict(out=A + 8),
               dict(qkv=A + 4), dict(wq=A + 4), dict(wk=A + 8), dict(cos=A + 4)):
        assert call(**kw) == INVALID, kw
    for rot in (0, 8, 24, 80):
        assert call(rot=rot) == UNSUPPORTED, rot
    assert call(n=0, out=None, qkv=None) == 0


def test_plan_refusals():
    L = lib()

    def call(table=A, start=A, lens=A, pos=A, slots=A, counts=A, cached=A, new=A, free=A, n_free=1, n_req=1, width=1,
             bs=16, n=1):
        return L.tl_paged_plan(table, start, lens, pos, slots, counts, cached, new, free, n_free, n_req, width, bs, n,
                               None)

    for kw in (dict(table=None), dict(start=None), dict(lens=None), dict(pos=None), dict(slots=None), dict(counts=None),
               dict(cached=None), dict(new=None), dict(free=None), dict(width=0), dict(width=1 << 31),
               dict(n_req=1 << 20, width=1 << 11), dict(n=1 << 31), dict(n_free=1 << 31)):
        assert call(**kw) == INVALID, kw
    for bs in (0, 4, 24, 512):
        assert call(bs=bs) == UNSUPPORTED


def test_sample_refusals():
    L = lib()

    def call(out=A, x=A, dtype=0, stride=100, rows=1, n=100, r=A, t=A):
        return L.tl_sample_rows(out, x, dtype, stride, rows, n, r, t, None, None, None, None)

    for kw in (dict(out=None), dict(x=None), dict(r=None), dict(t=None), dict(dtype=5), dict(n=0), dict(stride=99),
               dict(n=1 << 22, stride=1 << 22), dict(rows=1 << 31), dict(x=A + 2)):
        assert call(**kw) == INVALID, kw
    assert call(rows=0, out=None) == 0


def test_python_checks_refuse_before_the_library():
    torch = pytest.importorskip("torch")
    from torchless_b200 import ops
    i = torch.zeros(2, dtype=torch.int32)
    kc = torch.zeros(3, 2, 16, 64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_plan(torch.zeros(2, 3, dtype=torch.int32), i, i, i, 16, 4)
    with pytest.raises(ValueError, match="block_table"):
        ops.paged_plan(i, i, i, i, 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_attention(kc[0], kc[0], kc, kc, i, i, i)
    with pytest.raises(ValueError, match="layout"):
        ops.paged_attention(kc[0], kc[0], kc, kc[:2], i, i, i)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample_rows(torch.zeros(2, 5), i, i)
    with pytest.raises(ValueError, match="logits"):
        ops.sample_rows(torch.zeros(5), i, i)
