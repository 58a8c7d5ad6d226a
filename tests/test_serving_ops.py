"""Schemas and fake kernels of the serving operators without a counterpart in the
reference, and what the C entry of extend_block_tables refuses (no GPU)."""

import ctypes

import pytest
import torch

import gaudirt_amd
from gaudirt_amd import capi

ATTENTION = ("Tensor query, Tensor key, Tensor value, Tensor(a!) key_pool, Tensor(b!) value_pool, "
             "__torch__.torch.classes.gaudirt.PagedMetadata metadata, ")


@pytest.fixture(scope="module", autouse=True)
def extension():
    gaudirt_amd.load_extension()


@pytest.mark.parametrize("name,schema", [
    ("shared_prefix_attn", ATTENTION + "int[] group_rows, int[] group_prefix, int head_dim, float scale, "
     "float softcap=0., int sliding_window=-1) -> Tensor"),
    ("paged_attn_alibi", ATTENTION + "Tensor slopes, int head_dim, float scale, float softcap=0., int sliding_window=-1) "
     "-> Tensor"),
    ("extend_block_tables", "Tensor(a!) block_tables, Tensor(b!)? mapping, Tensor requests, Tensor prefixes, "
     "Tensor lengths, Tensor free_pages, Tensor? free_head, Tensor? parents, int page_size, int slots, int max_rows) -> "
     "(Tensor, Tensor, Tensor, Tensor, Tensor)"),
])
def test_schemas(name, schema):
    assert str(getattr(torch.ops.gaudirt, name).default._schema) == f"gaudirt::{name}({schema}"


@pytest.mark.parametrize("with_map", [True, False])
def test_fake_tables(with_map):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
        i64 = lambda *s: torch.empty(s, dtype=torch.int64, device="cuda")  # noqa: E731
        got = torch.ops.gaudirt.extend_block_tables(i32(9, 32), i32(9, 512) if with_map else None, i32(4), i64(4), i64(4),
                                                    i64(100), None, None, 16, 4096, 70)
        assert [(tuple(t.shape), t.dtype, t.device.type) for t in got] == [
            ((70,), torch.int32, "cuda")] * 3 + [((4,), torch.int64, "cuda"), ((4,), torch.int32, "cuda")]


def extend_params():
    p = capi.ExtendParams()
    fake = 1 << 20  # never dereferenced: every refused call returns before a launch
    for field in ("block_tables", "mapping", "seq_requests", "prefixes", "lengths", "parents", "free_pages", "free_head",
                  "out_locations", "out_requests", "out_positions", "out_lengths", "counts"):
        setattr(p, field, fake)
    p.requests, p.pages, p.context = 8, 32, 512
    p.free_count, p.batch, p.page_size, p.slots, p.max_rows = 100, 4, 16, 4096, 64
    return p


@pytest.mark.parametrize("change,message", [
    ({"struct_size": 8}, "struct_size"), ({"batch": -1}, "8192"), ({"batch": 8193}, "8192"), ({"requests": 0}, "table size"),
    ({"pages": 0}, "table size"), ({"requests": 1 << 20, "pages": 1 << 12}, "table size"), ({"context": 0}, "map size"),
    ({"requests": 1 << 20, "context": 1 << 12}, "map size"), ({"page_size": 0}, "page_size"), ({"page_size": 48}, "page_size"),
    ({"page_size": 1 << 21}, "page_size"), ({"slots": 0}, "out of range"), ({"slots": 1 << 31}, "out of range"),
    ({"free_count": -1}, "out of range"), ({"max_rows": -1}, "out of range"), ({"max_rows": (1 << 30) + 1}, "out of range"),
    ({"block_tables": None}, "null pointer"), ({"counts": None}, "null pointer"), ({"lengths": None}, "null pointer"),
    ({"out_lengths": None}, "null pointer"), ({"free_pages": None}, "null pointer"), ({"out_positions": None}, "null pointer"),
])
def test_extend_refuses(change, message):
    p = extend_params()
    for field, value in change.items():
        setattr(p, field, value)
    assert capi.load().gk_extend_block_tables(ctypes.byref(p), None) == capi.GK_ERR_INVALID_ARGUMENT
    assert message in capi.load().gk_last_error().decode()


def test_extend_refuses_null():
    assert capi.load().gk_extend_block_tables(None, None) == capi.GK_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("out,inputs,offset,length", [
    ("counts", "free_head", 12, 4), ("counts", "free_head", 0, 4), ("out_lengths", "prefixes", 0, 8),
    ("out_lengths", "prefixes", -28, 8), ("out_lengths", "lengths", 12, 4),
])
def test_extend_refuses_outputs_over_inputs(out, inputs, offset, length):
    p = extend_params()
    for i, (field, kind) in enumerate(p._fields_):
        if kind is ctypes.c_void_p:
            setattr(p, field, (1 << 20) + (i << 12))
    p.lengths_int64 = length == 8
    setattr(p, inputs, getattr(p, out) + offset)
    assert capi.load().gk_extend_block_tables(ctypes.byref(p), None) == capi.GK_ERR_INVALID_ARGUMENT
    assert "overlap" in capi.load().gk_last_error().decode()
