"""Host-side validation of the entry points for prompts and drafted tokens over paged keys and values (no GPU needed)."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from asterq import _lib

REPO = Path(__file__).resolve().parent.parent
STRUCTS = {"asterq_rows_attention_params": _lib.RowsAttentionParams, "asterq_kv_append_normed_params": _lib.KvAppendNormedParams,
           "asterq_kv_keep_params": _lib.KvKeepParams, "asterq_kv_copy_params": _lib.KvCopyParams,
           "asterq_verify_params": _lib.VerifyParams}


def test_mirrors_match_the_c_compiler(tmp_path):
    """Sizes, field offsets and the packed form of the parameter structs equal the C compiler's layout."""
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "asterq.h"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append(f'  printf("{name} sizeof %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, value = line.split()
        cls = STRUCTS[name]
        assert int(value) == (ctypes.sizeof(cls) if field == "sizeof" else getattr(cls, field).offset), (name, field)
    for cls in STRUCTS.values():
        pack = _lib.packer(cls)
        assert pack.size == ctypes.sizeof(cls)
        values = [i + 1 for i in range(len(cls._fields_))]
        got = cls.from_buffer_copy(pack.pack(*values))
        assert [getattr(got, f) for f, _ in cls._fields_] == values


def test_header_fields_match_the_mirrors():
    text = (REPO / "include" / "asterq.h").read_text()
    for name, cls in STRUCTS.items():
        body = re.sub(r"/\*.*?\*/", "", text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")], flags=re.S)
        fields = [re.sub(r"[*\s]", "", f.split()[-1]) for stmt in body.split("{", 1)[1].split(";") if stmt.strip()
                  for f in stmt.split(",")]
        assert fields == [f for f, _ in cls._fields_]


def _call(fn, cls, fields):
    p = cls()
    for k, v in fields.items():
        setattr(p, k, v)
    return getattr(_lib.load(), fn)(ctypes.byref(p), None)


BAD, NO, ODD, SMALL = (_lib.ASTERQ_ERR_INVALID_ARGUMENT, _lib.ASTERQ_ERR_UNSUPPORTED, _lib.ASTERQ_ERR_MISALIGNED,
                       _lib.ASTERQ_ERR_WORKSPACE)
ROWS = dict(dtype=_lib.DTYPE_F16, out_dtype=_lib.DTYPE_F16, n_seqs=1, n_heads=4, n_kv_heads=2, head_dim=64, page_tokens=16,
            max_pages=1, softmax_scale=1.0, n_rows=1, n_pages=1, q_row_stride=256, q_head_stride=64, q=16, k_pool=16,
            v_pool=16, page_table=16, lengths=16, row_offsets=16, out=16, workspace=16, workspace_bytes=1 << 30)
NORMED = dict(dtype=_lib.DTYPE_BF16, norm_dtype=_lib.DTYPE_F32, n_seqs=1, n_heads=4, n_kv_heads=2, head_dim=64, rotary_dim=64,
              page_tokens=16, max_pages=1, norm_eps=1e-6, n_rows=1, n_pages=1, n_positions=8, q_row_stride=256,
              q_head_stride=64, k_row_stride=128, k_head_stride=64, v_row_stride=128, v_head_stride=64, q=16, k=16, v=16,
              q_norm=16, k_norm=16, cos=16, sin=16, page_table=16, lengths=16, row_offsets=16, q_out=16, k_pool=16, v_pool=16)
POOLS = (ctypes.c_void_p * 2)(16, 32)
HOLE = (ctypes.c_void_p * 2)(16, 0)
KEEP = dict(dtype=_lib.DTYPE_BF16, n_layers=2, n_seqs=1, n_kv_heads=2, head_dim=64, page_tokens=16, max_pages=1, n_rows=1,
            n_pages=1, k_pools=ctypes.addressof(POOLS), v_pools=ctypes.addressof(POOLS), page_table=16, lengths=16,
            row_offsets=16, kept=16, n_kept=16)
COPY = dict(dtype=_lib.DTYPE_F16, n_layers=2, n_kv_heads=2, head_dim=64, page_tokens=16, n_pairs=1, n_pages=2,
            k_pools=ctypes.addressof(POOLS), v_pools=ctypes.addressof(POOLS), pairs=16)
VERIFY = dict(dtype=_lib.DTYPE_F32, n_seqs=1, vocab=8, n_rows=1, target_stride=8, target=16, tokens=16, row_offsets=16,
              accept=16, sample=16, kept=16, n_kept=16, next_token=16)


@pytest.mark.parametrize("kw,status", [
    (dict(n_rows=-1), BAD), (dict(n_seqs=-1), BAD), (dict(n_kv_heads=0), BAD), (dict(n_heads=3), BAD), (dict(page_tokens=0), BAD),
    (dict(window=-1), BAD), (dict(sink=-1), BAD), (dict(dtype=_lib.DTYPE_F32), NO), (dict(out_dtype=_lib.DTYPE_BF16), NO),
    (dict(head_dim=80), NO), (dict(page_tokens=24), NO), (dict(n_heads=258, n_kv_heads=2), NO), (dict(n_pages=1 << 31), NO),
    (dict(max_pages=1 << 28), NO), (dict(n_rows=1 << 31), NO), (dict(q=0), BAD), (dict(lengths=0), BAD), (dict(row_offsets=0), BAD),
    (dict(out=0), BAD), (dict(page_table=0), BAD), (dict(k_pool=0), BAD), (dict(workspace=0), BAD), (dict(q=24), ODD),
    (dict(out=8), ODD), (dict(q_row_stride=252), ODD), (dict(q_head_stride=0), NO), (dict(q_row_stride=-256), NO),
])
def test_rows_attention_refuses(kw, status):
    assert _call("asterq_rows_attention", _lib.RowsAttentionParams, ROWS | kw) == status
    assert b"rows_attention" in _lib.load().asterq_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(n_rows=-1), BAD), (dict(page_tokens=0), BAD), (dict(dtype=_lib.DTYPE_F32), NO), (dict(norm_dtype=_lib.DTYPE_F16), NO),
    (dict(head_dim=72), NO), (dict(head_dim=528), NO), (dict(rotary_dim=24), NO), (dict(rotary_dim=80), NO), (dict(k=0), BAD),
    (dict(cos=0), BAD), (dict(q_out=0), BAD), (dict(norm_eps=-1.0), BAD), (dict(norm_eps=float("nan")), BAD), (dict(v=8), ODD),
    (dict(k_row_stride=4), ODD),
])
def test_append_normed_refuses(kw, status):
    assert _call("asterq_kv_append_normed", _lib.KvAppendNormedParams, NORMED | kw) == status
    assert b"kv_append_normed" in _lib.load().asterq_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(n_layers=-1), BAD), (dict(n_seqs=-1), BAD), (dict(n_rows=-1), BAD), (dict(dtype=_lib.DTYPE_F32), NO),
    (dict(head_dim=12), NO), (dict(k_pools=0), BAD), (dict(kept=0), BAD), (dict(page_table=0), BAD), (dict(n_seqs=65536), NO),
    (dict(v_pools=ctypes.addressof(HOLE)), BAD),
])
def test_keep_refuses(kw, status):
    assert _call("asterq_kv_keep", _lib.KvKeepParams, KEEP | kw) == status
    assert b"kv_keep" in _lib.load().asterq_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(n_pairs=-1), BAD), (dict(n_pages=-1), BAD), (dict(dtype=7), NO), (dict(head_dim=12), NO), (dict(pairs=0), BAD),
    (dict(pairs=4), ODD), (dict(page_tokens=1 << 30, head_dim=64), NO),
])
def test_copy_refuses(kw, status):
    assert _call("asterq_kv_copy_pages", _lib.KvCopyParams, COPY | kw) == status
    assert b"kv_copy_pages" in _lib.load().asterq_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(n_seqs=-1), BAD), (dict(vocab=0), BAD), (dict(n_rows=-1), BAD), (dict(dtype=5), NO), (dict(target=0), BAD),
    (dict(tokens=0), BAD), (dict(accept=0), BAD), (dict(sample=0), BAD), (dict(kept=0), BAD), (dict(row_offsets=0), BAD),
    (dict(target_stride=-8), BAD), (dict(n_seqs=1 << 28), NO),
])
def test_verify_refuses(kw, status):
    assert _call("asterq_verify_drafts", _lib.VerifyParams, VERIFY | kw) == status
    assert b"verify_drafts" in _lib.load().asterq_last_error()


@pytest.mark.parametrize("fn,cls,fields,empty", [
    ("asterq_rows_attention", _lib.RowsAttentionParams, ROWS, dict(n_rows=0)),
    ("asterq_rows_attention", _lib.RowsAttentionParams, ROWS, dict(n_seqs=0)),
    ("asterq_kv_append_normed", _lib.KvAppendNormedParams, NORMED, dict(n_rows=0)),
    ("asterq_kv_keep", _lib.KvKeepParams, KEEP, dict(n_seqs=0)),
    ("asterq_kv_copy_pages", _lib.KvCopyParams, COPY, dict(n_pairs=0)),
    ("asterq_verify_drafts", _lib.VerifyParams, VERIFY, dict(n_seqs=0)),
])
def test_nothing_to_do_is_no_error(fn, cls, fields, empty):
    assert _call(fn, cls, fields | empty) == _lib.ASTERQ_OK


def test_null_parameters_are_refused():
    for fn in ("asterq_rows_attention", "asterq_kv_append_normed", "asterq_kv_keep", "asterq_kv_copy_pages", "asterq_verify_drafts"):
        assert getattr(_lib.load(), fn)(None, None) == BAD
