"""The speculative-step entry points without a GPU: the C header against the ctypes mirrors, what the functions refuse before they reach the device, and
the masks' layout."""
import ctypes
import re
import subprocess
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
ROOT = Path(__file__).resolve().parents[1]
HEADER = (ROOT / "include" / "dsv4_speculative.h").read_text()
STRUCTS = {"Dsv4HcaTreeDecodeParams": "HcaTreeDecodeParams", "Dsv4KvPagesParams": "KvPagesParams", "Dsv4SampleParams": "SampleParams"}
LAUNCHES = {"dsv4_hca_tree_decode_fwd": "HcaTreeDecodeParams", "dsv4_kv_pages_copy": "KvPagesParams", "dsv4_kv_pages_fork": "KvPagesParams",
            "dsv4_kv_pages_free": "KvPagesParams", "dsv4_kv_pages_compact": "KvPagesParams", "dsv4_kv_entries_move": "KvPagesParams", "dsv4_sample_fwd": "SampleParams"}
INVALID = 1            # cudaErrorInvalidValue


@pytest.fixture(scope="module")
def lib():
    from dsv4_attn_b200 import _lib, build
    build.build(quiet=True)
    return _lib


def test_every_function_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", HEADER, flags=re.S)
    names = set(re.findall(r"^\s*(?:int64_t|int|void)\s+(\w+)\s*\(", text, flags=re.M))
    assert names == set(LAUNCHES) | {"dsv4_hca_tree_rows_bytes"}
    for name in names:
        assert hasattr(lib.LIB, name)


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
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dsv4_speculative.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(tmp_path / "s")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


@pytest.mark.parametrize("name", sorted(LAUNCHES))
def test_null_and_empty_parameters_are_refused(lib, name):
    f = getattr(lib.LIB, name)
    assert f(None, None) == INVALID
    assert f(ctypes.byref(getattr(lib, LAUNCHES[name])()), None) == INVALID


def test_sample_refuses_sizes_and_types(lib):
    def call(**kw):
        p = lib.SampleParams(N=2, V=100, dtype=0, stride_n=100, logits=4096, u=4096, token=4096)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.LIB.dsv4_sample_fwd(ctypes.byref(p), None)
    for bad in (dict(N=-1), dict(V=0), dict(V=(1 << 22) + 1, stride_n=1 << 23), dict(stride_n=99), dict(logits=None), dict(u=None), dict(token=None), dict(dtype=3),
                dict(dtype=-1), dict(logits=4098), dict(dtype=1, logits=4097)):
        assert call(**bad) == INVALID, bad
    assert call(N=0) == 0


def test_pages_refuse_sizes_and_pointers(lib):
    def call(name, **kw):
        p = lib.KvPagesParams(pool=4096, num_pages=8, layers=1, entries=8, B=2, max_pages=4, n=1, src=4096, dst=4096, block_table=4096, kv_len=4096, refs=4096,
                              new_table=4096, new_refs=4096, count=4096, scratch=4096)
        for k, v in kw.items():
            setattr(p, k, v)
        return getattr(lib.LIB, name)(ctypes.byref(p), None)
    bad = {"dsv4_kv_pages_copy": ("pool", "src", "dst"), "dsv4_kv_entries_move": ("pool", "src", "dst"), "dsv4_kv_pages_free": ("block_table", "kv_len", "refs", "src"),
           "dsv4_kv_pages_fork": ("pool", "block_table", "kv_len", "refs", "src", "dst"),
           "dsv4_kv_pages_compact": ("pool", "block_table", "refs", "new_table", "new_refs", "count", "scratch")}
    for name, pointers in bad.items():
        for field in pointers:
            assert call(name, **{field: None}) == INVALID, (name, field)
    for name in ("dsv4_kv_pages_copy", "dsv4_kv_pages_fork", "dsv4_kv_pages_compact"):
        for sizes in (dict(num_pages=0), dict(num_pages=1 << 31), dict(layers=0), dict(pool=4104)):
            assert call(name, **sizes) == INVALID, (name, sizes)
    assert call("dsv4_kv_entries_move", entries=0) == INVALID
    for name in ("dsv4_kv_pages_copy", "dsv4_kv_pages_fork", "dsv4_kv_pages_free", "dsv4_kv_entries_move"):
        assert call(name, n=-1) == INVALID
        assert call(name, n=0) == 0


def test_tree_refuses_sizes_and_pointers(lib):
    def call(**kw):
        p = lib.HcaTreeDecodeParams(B=2, T=3, H=8, max_pages=4, win_cap=8, mask_words=1, num_splits=1, sm_scale=0.1, num_pages=8, q=4096, kv_pool=4096, block_table=4096,
                                    kv_len=4096, win_pool=4096, win_len=4096, tree_mask=4096, out=4096)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.LIB.dsv4_hca_tree_decode_fwd(ctypes.byref(p), None)
    for bad in (dict(B=0), dict(T=0), dict(H=0), dict(B=1 << 20, T=1 << 12, H=1), dict(max_pages=0), dict(win_cap=-1), dict(mask_words=-1), dict(num_splits=-1), dict(num_splits=2),
                dict(num_splits=0), dict(sm_scale=0.0), dict(sm_scale=float("nan")), dict(num_pages=0), dict(q=None), dict(kv_pool=None), dict(block_table=None),
                dict(kv_len=None), dict(win_pool=None), dict(win_len=None), dict(tree_mask=None), dict(out=None), dict(kv_pool=4104), dict(out=4100),
                dict(rows=4096, rows_bytes=100), dict(rows=4112, rows_bytes=1 << 30)):
        assert call(**bad) == INVALID, bad


def test_tree_rows_bytes(lib):
    f = lib.LIB.dsv4_hca_tree_rows_bytes
    assert f(1, 1, 0) == 64 * 1152 + 8
    assert f(3, 2, 1) == 3 * 192 * 1152 + 3 * 24           # whole tiles of 64 entries
    assert f(0, 1, 1) == f(1, 0, 1) == f(1, 1, -1) == 0
    assert f(1 << 14, 1 << 12, 0) == 0                     # more rows than a coordinate of 32 bits counts


@pytest.mark.parametrize("W", [1, 31, 32, 33, 100])
def test_pack_tree_mask(W):
    from dsv4_attn_b200 import layout
    sees = torch.rand(2, 3, W, generator=torch.Generator().manual_seed(W)) < 0.5
    words = layout.pack_tree_mask(sees)
    assert words.dtype == torch.int32 and words.shape == (2, 3, (W + 31) // 32)
    for b in range(2):
        for t in range(3):
            for w in range(32 * words.shape[2]):
                bit = int(words[b, t, w // 32]) >> (w % 32) & 1
                assert bit == (int(sees[b, t, w]) if w < W else 0)
    with pytest.raises(ValueError):
        layout.pack_tree_mask(sees.float())


def test_tree_sees_ancestors_and_its_window():
    from dsv4_attn_b200 import layout
    parents = torch.tensor([[-1, 0, 0, 2, -1]])
    sees = layout.tree_sees(parents, 6)[0]
    draft = [[0], [0, 1], [0, 2], [0, 2, 3], [4]]
    for t, ancestors in enumerate(draft):
        assert sees[t, 6:].nonzero()[:, 0].tolist() == ancestors
        # as many committed tokens as complete a window of 6
        assert sees[t, :6].nonzero()[:, 0].tolist() == list(range(len(ancestors), 6))
