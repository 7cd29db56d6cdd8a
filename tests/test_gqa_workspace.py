"""What the workspace of a call over K and V pages goes by.  No GPU needed."""
import ctypes

import pytest

torch = pytest.importorskip("torch")
BF16, E4M3 = 1, 3
GIB = 1 << 30


@pytest.fixture(scope="module")
def lib():
    from dsv4_attn_b200 import _lib, build
    build.build(quiet=True)
    return _lib


def size(lib, **kw):
    p = dict(B=8, T=1, Hkv=8, G=4, D=128, max_pages=2048, q_dtype=BF16, kv_dtype=BF16, sm_scale=0.1, rows=8, num_pages=8, q_stride_b=4096, q_stride_t=4096, q_stride_h=128)
    return lib.LIB.dsv4_gqa_workspace_bytes(ctypes.byref(lib.GqaParams(**{**p, **kw})))


PROMPT = dict(T=0, rows=16_000, q_start=4096, kv_dtype=E4M3)


def test_copies_for_prompts_over_8_bits(lib):
    # a table's capacity, 512 bytes an entry and head; up to 4 GiB
    one = 2048 * 64 * 8 * 128 * 4
    for B in (1, 2, 8):
        assert 0 <= size(lib, **PROMPT, B=B) - B * one < 16 << 20
    for kw in (dict(B=16), dict(B=500), dict(B=1, max_pages=16384), dict(B=3, max_pages=100_000), dict(B=2, max_pages=5000, Hkv=64)):
        assert one < size(lib, **{**PROMPT, **kw}) <= 4 * GIB + (16 << 20), kw
    # or the longest length
    for B in (1, 16, 64):
        assert 0 <= size(lib, **PROMPT, B=B, max_len=2000) - B * 2048 * 8 * 128 * 4 < 16 << 20
    assert size(lib, **PROMPT, max_len=1 << 20) == size(lib, **PROMPT)


def test_scores_for_weights(lib):
    # a score for every row and entry, and a denominator a row
    rows, room = 8 * 32, 2048 * 64
    kw = dict(weights=4096, weight_stride=room)
    assert size(lib, **kw) - size(lib) == rows * room * 4 + rows * 4
    for n, entries in ((64, 64), (1000, 1024), (room - 1, room), (room, room), (1 << 30, room)):
        assert size(lib, **kw, max_len=n) - size(lib, max_len=n) == rows * entries * 4 + rows * 4
