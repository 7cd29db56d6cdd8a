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


@pytest.mark.parametrize("call", [dict(), dict(T=5, G=16, rows=40), dict(T=5, G=16, rows=40, kv_dtype=E4M3), PROMPT, dict(PROMPT, kv_dtype=BF16), dict(weights=4096, weight_stride=1 << 20)])
def test_nothing_else(lib, call):
    """What the header names, and no other field: buffers, scales, sink, factor, pool and status may follow later."""
    n = size(lib, **call)
    assert n > 0
    later = dict(q=4096, k_pool=4096, v_pool=4096, block_table=4096, kv_len=4096, k_scale=4096, v_scale=4096, attn_sink=4096, out=4096, lse=4096, workspace=4096, workspace_bytes=1, status=4096,
                 sm_scale=3.0, num_pages=1000, q_dtype=2, q_stride_t=8192, q_stride_h=256, q_stride_b=1 << 20)
    for k, v in later.items():
        assert size(lib, **{**call, k: v}) == n, k


def test_types_and_strides_of_zero(lib):
    assert size(lib, **PROMPT) > size(lib, **{**PROMPT, "kv_dtype": BF16})
    # rows that are shared: other kernels, whose parts need room
    prompt = {**PROMPT, "kv_dtype": BF16}
    assert size(lib, **prompt, q_stride_t=0) > size(lib, **prompt) and size(lib, **prompt, q_stride_h=0) > size(lib, **prompt)
    many = dict(T=5, G=16, rows=40)
    assert len({size(lib, **many), size(lib, **many, q_stride_b=0)}) == 2
    assert size(lib, **many, kv_dtype=E4M3) == size(lib, **many, kv_dtype=E4M3, q_stride_b=0)
