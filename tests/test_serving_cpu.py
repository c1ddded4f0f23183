"""CPU tests of the serving operators: what the public functions refuse, what the C entry points refuse
before they touch a device, and the layout of their structures."""

import ctypes as C
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import piper_kernels_b200 as pk
from _serving import ListCache
from piper_kernels_b200 import _cabi, _ops

ROOT = Path(__file__).resolve().parents[1]


def rows(batch=2, heads=4, length=8, dim=64, dtype=torch.float16):
    return torch.zeros(batch, heads, length, dim, dtype=dtype)


def ints(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype)


def window(q=None, k=None, v=None, **kw):
    q, k = rows() if q is None else q, rows() if k is None else k
    return pk.window_attention(q, k, k if v is None else v, **{"window": 4, **kw})


def test_window_attention_refuses():
    for match, call in {
        "float16 or bfloat16": lambda: window(rows().float()),
        "shape": lambda: window(rows()[0]),
        "share a dtype": lambda: window(rows(dtype=torch.bfloat16)),
        "head dimensions 64 and 128": lambda: window(rows(dim=32), rows(dim=32)),
        "head dimensions must match": lambda: window(rows(dim=128)),
        "head dimension must be contiguous": lambda: window(torch.zeros(2, 4, 64, 64, dtype=torch.float16).transpose(2, 3)),
        "shapes must match": lambda: window(v=rows(length=7)),
        "equal batch": lambda: window(rows(batch=1)),
        "does not accept empty": lambda: window(rows(length=0)),
        "multiple of the key heads": lambda: window(rows(heads=6)),
        "window must be": lambda: window(window=0),
        "window must be an integer": lambda: window(window=2.5),
        "sinks must be": lambda: window(sinks=-1),
        "lengths must be int32 of shape": lambda: window(lengths=ints(3)),
        "lengths must be int32": lambda: window(lengths=ints(2, dtype=torch.int64)),
        "lengths must be contiguous": lambda: window(lengths=ints(4)[::2]),
        "finite and positive": lambda: window(scale=-1.0),
    }.items():
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="inference-only"):
        window(rows().requires_grad_())
    with pytest.raises(RuntimeError, match="no CPU path"):
        window()


def cache(**kw):
    return pk.PageCache(**{"batch": 2, "pages": 6, "page_size": 16, "kv_heads": 2, "head_dim": 64, "dtype": torch.float16, "device": "cpu", **kw})


def test_page_cache_refuses():
    c = cache(layers=2)
    for match, call in {
        "page_size must be one of": lambda: cache(page_size=24),
        "head dimensions 64 and 128": lambda: cache(head_dim=96),
        "pages must be positive": lambda: cache(pages=0),
        "max_length must be positive": lambda: cache(max_length=0),
        "float16, bfloat16 or int8": lambda: cache(dtype=torch.float32),
        "at most 4096": lambda: cache(batch=4097, max_length=16),
        "counts must be int32": lambda: c.extend(ints(2, dtype=torch.int64)),
        "counts must be int32 of shape": lambda: c.extend(ints(3)),
        "counts must be": lambda: c.extend(None),
        "parents must be int32": lambda: c.fork(ints(1)),
        "lengths must be int32": lambda: c.truncate(ints(2, 1)),
        "paths must be int32": lambda: c.compact(ints(2), ints(2)),
        "paths must be int32 of shape": lambda: c.compact(ints(2, 0), ints(2)),
        "last dimension must be contiguous": lambda: c.compact(ints(3, 2).T, ints(2)),
        "layer must be in": lambda: c.write(rows(heads=2), rows(heads=2), layer=2),
        r"\[layers, batch": lambda: c.write(rows(heads=2), rows(heads=2)),
        "must have shape": lambda: c.write(rows(heads=4), rows(heads=4), layer=0),
        "must match": lambda: c.write(rows(heads=2), rows(heads=2, length=9), layer=0),
        "share a dtype": lambda: c.write(rows(heads=2, dtype=torch.bfloat16), rows(heads=2, dtype=torch.bfloat16), layer=0),
        "empty rows": lambda: c.write(rows(heads=2, length=0), rows(heads=2, length=0), layer=0),
        "count must be": lambda: c.read(ints(2), 0),
        "reads as": lambda: c.read(ints(2), 1, dtype=torch.int8),
        "first must be int32": lambda: c.read(ints(1), 1),
    }.items():
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.extend(ints(2))
    with pytest.raises(RuntimeError, match="no CPU path"):
        c.read(ints(2), 4)
    with pytest.raises(RuntimeError, match="inference-only"):
        c.write(rows(heads=2).requires_grad_(), rows(heads=2), layer=0)


def test_page_cache_from_tensors_refuses():
    c = cache(dtype=torch.int8)
    good = {n: getattr(c, n) for n in ("keys", "values", "table", "lengths", "starts", "uses", "key_scales", "value_scales")}
    same = pk.PageCache.from_tensors(**good)
    assert same.keys is c.keys and same.max_length == c.max_length == 96 and same.dtype is torch.int8
    for name, wrong in {"values": good["values"][:, :5], "table": good["table"].long(), "lengths": ints(3), "starts": None, "uses": ints(5),
                        "key_scales": None, "value_scales": good["value_scales"].double(), "keys": good["keys"].transpose(1, 2)}.items():
        with pytest.raises(ValueError):
            pk.PageCache.from_tensors(**{**good, name: wrong})
    with pytest.raises(ValueError, match="belongs to an int8 cache"):
        pk.PageCache.from_tensors(**{**good, "keys": good["keys"].half(), "values": good["values"].half()})


def test_cache_attention_refuses():
    c, eight = cache(), cache(dtype=torch.int8)
    q = rows(length=3)
    for match, call in {
        "shape": lambda: pk.cache_attention(q[0], c),
        "share a dtype": lambda: pk.cache_attention(q.to(torch.bfloat16), c),
        "one query row per sequence": lambda: pk.cache_attention(q[:1], c),
        "empty queries": lambda: pk.cache_attention(q[:, :, :0], c),
        "multiple of the cache's heads": lambda: pk.cache_attention(q[:, :3], c),
        "head dimensions must match": lambda: pk.cache_attention(rows(dim=128), c),
        "layer must be in": lambda: pk.cache_attention(q, c, layer=1),
        "window must be": lambda: pk.cache_attention(q, c, window=0),
        "sinks must be": lambda: pk.cache_attention(q, c, sinks=True),
        "tree must be int32 of shape": lambda: pk.cache_attention(q, c, tree=ints(2, 4)),
        "tree must be int32": lambda: pk.cache_attention(q, c, tree=ints(3, dtype=torch.int64)),
        "at most 64 tokens": lambda: pk.cache_attention(rows(length=65), c, tree=ints(65)),
        "tree's last dimension": lambda: pk.cache_attention(q, c, tree=ints(3, 2).T),
        "finite and positive": lambda: pk.cache_attention(q, c, scale=float("nan")),
    }.items():
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="inference-only"):
        pk.cache_attention(q.clone().requires_grad_(), c)
    for good in (c, eight):
        with pytest.raises(RuntimeError, match="no CPU path"):
            pk.cache_attention(q, good, tree=ints(3))


def test_structures_match_the_header(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    pairs = {"pk_window_problem": _cabi.PkWindowProblem, "pk_cache": _cabi.PkCache, "pk_cache_query": _cabi.PkCacheQuery}
    src = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT}/include/piper_b200.h"', "int main(void){"]
    want = []
    for name, mirror in pairs.items():
        src.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(mirror))
        for field, *_ in mirror._fields_:
            src.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(mirror, field).offset)
    (tmp_path / "layout.c").write_text("\n".join([*src, "return 0;}"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "layout"), str(tmp_path / "layout.c")], check=True)
    out = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(x) for x in out] == want


def window_problem(**over):
    p = _cabi.PkWindowProblem()
    p.batch, p.heads, p.kv_heads, p.q_len, p.kv_len, p.head_dim, p.dtype = 1, 4, 2, 10, 100, 128, _cabi.PK_BF16
    p.window, p.sinks, p.scale = 16, 0, 0.1
    p.q = p.k = p.v = 256
    p.q_stride = p.k_stride = p.v_stride = (C.c_int64 * 3)(51200, 12800, 128)
    for k, v in over.items():
        setattr(p, k, v)
    return p


def test_window_entry_refuses_before_the_device():
    lib, n = _cabi.lib(), C.c_uint64()
    assert lib.pk_window_workspace_bytes(C.byref(window_problem()), C.byref(n)) == _cabi.PK_OK and n.value > 0
    for over in (dict(batch=0), dict(heads=3), dict(kv_heads=0), dict(q_len=0), dict(kv_len=-1), dict(head_dim=96), dict(dtype=_cabi.PK_F32), dict(window=0),
                 dict(sinks=-1), dict(scale=0.0), dict(scale=float("inf")), dict(q=None), dict(kv_len=2**30)):
        assert lib.pk_window_workspace_bytes(C.byref(window_problem(**over)), C.byref(n)) == _cabi.PK_ERR_BAD_ARG, over
        assert lib.pk_last_error()
    assert lib.pk_window_workspace_bytes(C.byref(window_problem()), None) == _cabi.PK_ERR_BAD_ARG
    assert lib.pk_window_attention_fwd(C.byref(window_problem())) == _cabi.PK_ERR_BAD_ARG  # no output
    assert lib.pk_window_attention_fwd(C.byref(window_problem(out=256))) == _cabi.PK_ERR_WORKSPACE
    assert lib.pk_window_attention_fwd(C.byref(window_problem(out=256, workspace=256, workspace_bytes=16))) == _cabi.PK_ERR_WORKSPACE


def test_window_workspace_holds_rows_that_no_copy_map_describes():
    lib, n, more = _cabi.lib(), C.c_uint64(), C.c_uint64()
    lib.pk_window_workspace_bytes(C.byref(window_problem()), C.byref(n))
    for over in (dict(k=258), dict(v_stride=(C.c_int64 * 3)(51200, 12800, 129)), dict(k_stride=(C.c_int64 * 3)(51200, 12800, 0))):
        lib.pk_window_workspace_bytes(C.byref(window_problem(**over)), C.byref(more))
        assert more.value >= n.value + 2 * 100 * 128 * 2


def c_cache(**over):
    c = _cabi.PkCache()
    c.layers, c.pages, c.kv_heads, c.page_size, c.head_dim, c.batch, c.width, c.dtype = 2, 10, 2, 16, 64, 3, 4, _cabi.PK_F16
    for name in ("keys", "values", "table", "lengths", "starts", "uses", "refused", "scratch"):
        setattr(c, name, 256)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def test_cache_entries_refuse_before_the_device():
    lib, n = _cabi.lib(), C.c_uint64()
    strides = (C.c_int64 * 4)(0, 64, 64, 64)
    for over in (dict(layers=0), dict(pages=0), dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(head_dim=32), dict(batch=4097), dict(width=0),
                 dict(width=2**26), dict(dtype=_cabi.PK_F32), dict(dtype=_cabi.PK_I8), dict(keys=264), dict(table=None), dict(scratch=None),
                 dict(pages=2**30, layers=4)):
        c = C.byref(c_cache(**over))
        assert lib.pk_cache_extend(c, 256) == _cabi.PK_ERR_BAD_ARG, over
        assert lib.pk_cache_truncate(c, 256) == lib.pk_cache_fork(c, 256) == lib.pk_cache_compact(c, 256, 4, 4, 256) == _cabi.PK_ERR_BAD_ARG
        assert lib.pk_cache_write(c, 0, 256, 256, strides, strides, _cabi.PK_F16, 3) == lib.pk_cache_read(c, 0, 256, 3, 256, 256, _cabi.PK_F16) == _cabi.PK_ERR_BAD_ARG
    assert lib.pk_cache_extend(None, 256) == _cabi.PK_ERR_BAD_ARG
    assert lib.pk_cache_maps(C.byref(c_cache(page_size=8)), 64) == lib.pk_cache_maps(C.byref(c_cache()), None) == lib.pk_cache_maps(C.byref(c_cache()), 72) == _cabi.PK_ERR_BAD_ARG
    query = _cabi.PkCacheQuery()

    def ask(cache=None, **over):
        query.heads, query.tokens, query.layer, query.dtype, query.window, query.sinks, query.scale, query.q, query.tree = 4, 5, 1, _cabi.PK_F16, 0, 0, 0.1, 256, None
        for k, v in over.items():
            setattr(query, k, v)
        return lib.pk_cache_attention_workspace_bytes(C.byref(cache or c_cache()), C.byref(query), C.byref(n))

    assert ask() == _cabi.PK_OK and n.value > 0
    assert ask(c_cache(dtype=_cabi.PK_I8, key_scales=256, value_scales=256), dtype=_cabi.PK_BF16) == _cabi.PK_OK
    for over in (dict(heads=3), dict(heads=0), dict(tokens=0), dict(layer=2), dict(layer=-1), dict(dtype=_cabi.PK_BF16), dict(dtype=_cabi.PK_I8), dict(window=-1),
                 dict(sinks=-1), dict(scale=-1.0), dict(q=None), dict(tree=256, tokens=65)):
        assert ask(**over) == _cabi.PK_ERR_BAD_ARG, over
    assert ask() == _cabi.PK_OK
    assert lib.pk_cache_attention_fwd(C.byref(c_cache()), C.byref(query)) == _cabi.PK_ERR_BAD_ARG  # no output
    query.out = 256
    assert lib.pk_cache_attention_fwd(C.byref(c_cache()), C.byref(query)) == _cabi.PK_ERR_WORKSPACE


def test_fake_kernel_of_window_attention():
    q = torch.empty(2, 4, 5, 64, dtype=torch.float16, device="meta").permute(1, 0, 2, 3)
    out = _ops.window_attention_op(q, q, q, None, 3, 0, 0.1)
    assert out.shape == q.shape and out.is_contiguous() and out.dtype == q.dtype


def test_list_model_of_the_cache():
    """The oracle itself, on a run whose result is written down here."""
    m = ListCache(3, 8, 16, 4)
    m.extend([20, 0, 5])
    assert m.own == [[0, 1], [], [2]] and m.start == [0, 0, 0] and m.length == [20, 0, 5]
    m.fork([0, 0, 2])
    assert m.own == [[0, 1], [0, 1], [2]] and m.uses()[:3] == [2, 2, 1]
    m.extend([1, 1, 1])  # both owners of page 1 grow: the first keeps it
    assert m.own == [[0, 1], [0, 3], [2]] and m.copied == [(1, 3, 4)]
    m.fork([0, 0, 0])
    m.extend([1, 0, 1])  # one owner does not grow: both that do get copies
    assert m.own == [[0, 2], [0, 1], [0, 3]]
    m.extend([60, 5, 0])
    assert m.refused == [1, 0, 0] and m.length == [22, 26, 22]
    m.extend([30, 10, 42])  # needs 2 + 1 + 2 of the pages 4, 5, 6, 7
    assert m.refused == [0, 0, 1] and m.own == [[0, 2, 4, 5], [0, 1, 6], [0, 3]]
    m.compact([[0, 3], [2, 1], []], [2, 2, 0])
    assert m.refused == [0, 1, 0] and m.length == [24, 36, 22] and m.own[0] == [0, 2]
    m.truncate([0, 16, 99])
    assert m.own == [[], [0], [0, 3]] and m.uses() == [2, 0, 0, 1, 0, 0, 0, 0]
