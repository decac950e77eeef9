"""Host-side validation of the paged K/V and linear-attention entry points (no GPU needed)."""
from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest

from asterq import _lib

REPO = Path(__file__).resolve().parent.parent
STRUCTS = {"asterq_kv_append_params": _lib.KvAppendParams, "asterq_paged_attention_params": _lib.PagedAttentionParams,
           "asterq_linear_params": _lib.LinearParams}


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


def _fill(cls, **kw):
    p = cls()
    for k, v in kw.items():
        setattr(p, k, v)
    return p


APPEND = dict(dtype=_lib.DTYPE_BF16, n_seqs=1, n_heads=4, n_kv_heads=2, head_dim=64, rotary_dim=64, page_tokens=16,
              max_pages=1, n_rows=1, n_pages=1, n_positions=8, q_row_stride=256, q_head_stride=64, k_row_stride=128,
              k_head_stride=64, v_row_stride=128, v_head_stride=64, q=16, k=16, v=16, cos=16, sin=16, page_table=16,
              lengths=16, row_offsets=16, q_out=16, k_pool=16, v_pool=16)
ATTEND = dict(dtype=_lib.DTYPE_F16, out_dtype=_lib.DTYPE_F16, n_rows=1, n_heads=4, n_kv_heads=2, head_dim=64,
              page_tokens=16, max_pages=1, n_pages=1, q_row_stride=256, q_head_stride=64, q=16, k_pool=16, v_pool=16,
              page_table=16, lengths=16, out=16, workspace=16, workspace_bytes=1 << 30)
LINEAR = dict(dtype=_lib.DTYPE_BF16, n_seqs=1, n_heads=2, dk=64, dv=64, n_slots=1, n_rows=1, q_row_stride=128,
              q_head_stride=64, k_row_stride=128, k_head_stride=64, v_row_stride=128, v_head_stride=64, q=16, k=16, v=16,
              log_decay=16, state=16, slots=16, out=16)


@pytest.mark.parametrize("kw,status", [
    (dict(n_rows=-1), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(page_tokens=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(n_kv_heads=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(dtype=_lib.DTYPE_F32), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(head_dim=72), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(head_dim=528), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(rotary_dim=24), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(rotary_dim=80), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(k=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(cos=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(q_out=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(lengths=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(v=24), _lib.ASTERQ_ERR_MISALIGNED),
    (dict(v_row_stride=129), _lib.ASTERQ_ERR_MISALIGNED),
])
def test_append_validation(kw, status):
    lib = _lib.load()
    assert lib.asterq_kv_append(ctypes.byref(_fill(_lib.KvAppendParams, **{**APPEND, **kw})), None) == status
    assert lib.asterq_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(n_rows=-1), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(n_heads=5), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(window=-1), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(sink=-1), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(n_new=-1), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(dtype=_lib.DTYPE_F32), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(out_dtype=_lib.DTYPE_BF16), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(head_dim=96), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(page_tokens=24), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(n_pages=1 << 31), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(max_pages=1 << 28), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(q=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(page_table=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(k_pool=24), _lib.ASTERQ_ERR_MISALIGNED),
    (dict(q=18), _lib.ASTERQ_ERR_MISALIGNED),
    (dict(q_row_stride=257), _lib.ASTERQ_ERR_MISALIGNED),
])
def test_attention_validation(kw, status):
    lib = _lib.load()
    assert lib.asterq_paged_attention(ctypes.byref(_fill(_lib.PagedAttentionParams, **{**ATTEND, **kw})), None) == status
    assert lib.asterq_last_error()


@pytest.mark.parametrize("kw,status", [
    (dict(n_rows=-1), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(n_heads=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(n_rows=2), _lib.ASTERQ_ERR_INVALID_ARGUMENT),  # two rows for one sequence of one token
    (dict(dk=96), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(dv=256), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(dtype=5), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(n_heads=1 << 20), _lib.ASTERQ_ERR_UNSUPPORTED),
    (dict(state=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(slots=0), _lib.ASTERQ_ERR_INVALID_ARGUMENT),
    (dict(state=8), _lib.ASTERQ_ERR_MISALIGNED),
    (dict(q_head_stride=60), _lib.ASTERQ_ERR_MISALIGNED),
])
def test_linear_validation(kw, status):
    lib = _lib.load()
    assert lib.asterq_linear_attention(ctypes.byref(_fill(_lib.LinearParams, **{**LINEAR, **kw})), None) == status
    assert lib.asterq_last_error()


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    assert lib.asterq_kv_append(ctypes.byref(_fill(_lib.KvAppendParams, **{**APPEND, "n_rows": 0})), None) == _lib.ASTERQ_OK
    assert lib.asterq_paged_attention(ctypes.byref(_fill(_lib.PagedAttentionParams, **{**ATTEND, "n_rows": 0})), None) == _lib.ASTERQ_OK
    assert lib.asterq_linear_attention(ctypes.byref(_fill(_lib.LinearParams, **{**LINEAR, "n_rows": 0})), None) == _lib.ASTERQ_OK
    for fn in (lib.asterq_kv_append, lib.asterq_paged_attention, lib.asterq_linear_attention):
        assert fn(None, None) == _lib.ASTERQ_ERR_INVALID_ARGUMENT


def test_cpu_tensors_are_refused():
    import torch

    from asterq.linear_attention import linear_attention_step
    from asterq.paged_kv import PagedKVPools

    x = torch.zeros(1, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        PagedKVPools(x, x)
    with pytest.raises(RuntimeError):
        linear_attention_step(torch.zeros(1, 1, 64, 64), torch.zeros(1, dtype=torch.int32), x[0], x[0], x[0], torch.zeros(1))
