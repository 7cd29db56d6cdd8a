"""The entry points over K and V pages without a GPU: the C header against the ctypes mirrors, and what the functions refuse before they reach the device."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
ROOT = Path(__file__).resolve().parents[1]
HEADER = (ROOT / "include" / "dsv4_gqa.h").read_text()
STRUCTS = {"Dsv4GqaParams": "GqaParams", "Dsv4GqaInsertParams": "GqaInsertParams", "Dsv4KvEvictParams": "KvEvictParams"}
LAUNCHES = {"dsv4_gqa_decode_fwd": "GqaParams", "dsv4_gqa_prefill_fwd": "GqaParams", "dsv4_gqa_insert": "GqaInsertParams", "dsv4_kv_evict": "KvEvictParams"}
INVALID = 1            # cudaErrorInvalidValue
BF16, F16, E4M3 = 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    from dsv4_attn_b200 import _lib, build
    build.build(quiet=True)
    return _lib


def test_every_function_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER, flags=re.S)
    names = set(re.findall(r"^\s*(?:int64_t|int|void)\s+(\w+)\s*\(", text, flags=re.M))
    assert names == set(LAUNCHES) | {"dsv4_gqa_workspace_bytes"}
    for name in names:
        assert hasattr(lib.LIB, name) and name in lib.EXPORTS


def test_struct_layouts(lib, tmp_path):
    assert set(re.findall(r"typedef struct (Dsv4\w+)", HEADER)) == set(STRUCTS)
    lines, want = [], []
    for cname, pyname in STRUCTS.items():
        mirror = getattr(lib, pyname)
        lines.append(f'printf("%zu\\n", sizeof({cname}));')
        want.append(ctypes.sizeof(mirror))
        for field, _ in mirror._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cname}, {field}));')
            want.append(getattr(mirror, field).offset)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dsv4_gqa.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


@pytest.mark.parametrize("name", sorted(LAUNCHES))
def test_null_and_empty_parameters_are_refused(lib, name):
    f = getattr(lib.LIB, name)
    assert f(None, None) == INVALID
    assert f(ctypes.byref(getattr(lib, LAUNCHES[name])()), None) == INVALID
    assert lib.LIB.dsv4_gqa_workspace_bytes(None) == -1


def attention(lib, **kw):
    p = lib.GqaParams(B=2, T=3, Hkv=2, G=4, D=128, max_pages=4, q_dtype=BF16, kv_dtype=BF16, sm_scale=0.1, rows=6, num_pages=8, q_stride_b=3 * 1024, q_stride_t=1024,
                      q_stride_h=128, q=4096, k_pool=4096, v_pool=4096, block_table=4096, kv_len=4096, out=4096, workspace=4096, workspace_bytes=1 << 40)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_attention_refuses_sizes_types_and_pointers(lib):
    common = (dict(B=0), dict(Hkv=0), dict(G=0), dict(G=1 << 20), dict(D=0), dict(D=96), dict(D=512), dict(max_pages=0), dict(max_pages=1 << 26), dict(window=-1), dict(first=-1),
              dict(q_dtype=0), dict(q_dtype=E4M3), dict(kv_dtype=F16), dict(kv_dtype=E4M3), dict(kv_dtype=E4M3, k_scale=4096), dict(sm_scale=0.0), dict(sm_scale=float("nan")),
              dict(num_pages=0), dict(num_pages=1 << 25), dict(q=None), dict(k_pool=None), dict(v_pool=None), dict(block_table=None), dict(kv_len=None), dict(out=None), dict(q=4104),
              dict(k_pool=4104), dict(v_pool=4104), dict(out=4104), dict(q_stride_t=1025), dict(q_stride_h=4), dict(workspace=None), dict(workspace=4097), dict(workspace_bytes=16))
    decode, prefill = lib.LIB.dsv4_gqa_decode_fwd, lib.LIB.dsv4_gqa_prefill_fwd
    for bad in (*common, dict(T=0), dict(T=-1), dict(rows=5), dict(q_start=4096), dict(weights=4096, weight_stride=255), dict(q_stride_b=12)):
        assert decode(ctypes.byref(attention(lib, **bad)), None) == INVALID, bad
    for bad in (*common, dict(rows=-1), dict(rows=0), dict(q_start=None), dict(weights=4096, weight_stride=256), dict(rows=1 << 40)):
        assert prefill(ctypes.byref(attention(lib, **dict(dict(q_start=4096), **bad))), None) == INVALID, bad


def test_workspace_bytes(lib):
    f = lib.LIB.dsv4_gqa_workspace_bytes
    n = f(ctypes.byref(attention(lib)))
    assert n > 0 and n % 128 == 0
    more = f(ctypes.byref(attention(lib, weights=4096, weight_stride=256)))
    assert more == n + 2 * 2 * 3 * 4 * 256 * 4 + 256                      # scores of every row, and their denominators
    assert f(ctypes.byref(attention(lib, D=100))) == -1


def test_insert_refuses(lib):
    def call(**kw):
        p = lib.GqaInsertParams(B=2, T=3, Hkv=2, D=64, max_pages=4, src_dtype=BF16, kv_dtype=BF16, rows=6, num_pages=8, k_stride_b=384, k_stride_t=128, k_stride_h=64,
                                v_stride_b=384, v_stride_t=128, v_stride_h=64, k=4096, v=4096, k_pool=4096, v_pool=4096, block_table=4096, insert_pos=4096)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.LIB.dsv4_gqa_insert(ctypes.byref(p), None)
    for bad in (dict(B=0), dict(T=-1), dict(rows=5), dict(rows=-1), dict(Hkv=0), dict(D=0), dict(D=60), dict(max_pages=0), dict(num_pages=0), dict(src_dtype=0), dict(src_dtype=E4M3),
                dict(kv_dtype=F16), dict(kv_dtype=E4M3), dict(k=None), dict(v=None), dict(k_pool=None), dict(v_pool=None), dict(block_table=None), dict(insert_pos=None), dict(k=4100),
                dict(v_pool=4100), dict(k_stride_t=100), dict(v_stride_h=1)):
        assert call(**bad) == INVALID, bad
    assert call(T=0, rows=0) == 0


def test_evict_refuses(lib):
    def call(**kw):
        p = lib.KvEvictParams(B=2, max_pages=4, pools=1, keep=10, num_pages=8, layers=2, block_table=4096, kv_len=4096, refs=4096, weights=4096, weight_stride=256, new_table=4096,
                              new_len=4096, new_refs=4096, new_weights=4096, kept=4096, scratch=4096)
        p.pool[0], p.entry_bytes[0] = 4096, 256
        for k, v in kw.items():
            if k in ("pool", "entry_bytes"):
                getattr(p, k)[0] = v
            else:
                setattr(p, k, v)
        return lib.LIB.dsv4_kv_evict(ctypes.byref(p), None)
    for bad in (dict(B=0), dict(B=70_000), dict(max_pages=0), dict(pools=5), dict(pools=-1), dict(pools=2), dict(keep=-1), dict(first=-1), dict(recent=-1), dict(num_pages=0),
                dict(num_pages=1 << 25), dict(layers=0), dict(weight_stride=255), dict(scratch=4104), dict(pool=None), dict(pool=4100), dict(entry_bytes=0), dict(entry_bytes=100),
                *(({k: None}) for k in ("block_table", "kv_len", "refs", "weights", "new_table", "new_len", "new_refs", "new_weights", "kept", "scratch"))):
        assert call(**bad) == INVALID, bad


def test_the_python_surface_names_what_is_wrong(lib):
    import dsv4_attn_b200 as d
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 64, 2, 64, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="q must be a cuda tensor"):
        d.gqa_decode(q, pool, pool, table, n, 0.1)
    with pytest.raises(ValueError, match="q_start must be a tensor"):
        d.gqa_prefill(q[0], None, pool, pool, table, n, 0.1)
    with pytest.raises(ValueError, match="k must be a cuda tensor"):
        d.gqa_insert(q, q, pool, pool, table, n)
    with pytest.raises(ValueError, match="block_table must be on cuda"):
        d.kv_evict((pool[None], pool[None]), table, n, n, torch.zeros(1, 128), 1)
