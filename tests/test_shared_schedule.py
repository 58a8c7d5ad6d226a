"""CPU tests of the shared-prefix work plan (gaudirt_amd/csrc/shared_schedule.hpp,
the code that gk_shared_prefix_list_build runs): tests/shared_schedule_test.cpp
built with g++, and the C entries' own checks (no GPU)."""

import ctypes
import pathlib
import subprocess

import numpy as np
import pytest

from gaudirt_amd import capi

ROOT = pathlib.Path(__file__).resolve().parent.parent


def test_plan_covers_every_key_once(tmp_path):
    exe = tmp_path / "shared_schedule_test"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=address,undefined", "-I",
                    str(ROOT / "gaudirt_amd" / "csrc"), str(ROOT / "tests" / "shared_schedule_test.cpp"), "-o",
                    str(exe)], check=True)
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
    assert run.stdout.strip() == "OK"


def build(first=(0, 1), rows=(1, 1), pos=(700, 900), group=(0, 0), prefix=(640,), heads=(32, 8, 128), window=-1,
          capacity=1 << 16, size=None, request=None):
    lib, as_i32 = capi.load(), lambda a: np.ascontiguousarray(a, dtype=np.int32)
    arrays = [as_i32(a) for a in (first, rows, pos, group)]
    prefix = as_i32(prefix)
    words, lst = np.full(max(capacity, 1), -7, dtype=np.int32), capi.SharedPrefixList()
    if size is not None:
        lst.struct_size = size
    ptr = lambda a: ctypes.c_void_p(a.ctypes.data)  # noqa: E731
    request = None if request is None else as_i32(request)
    rc = lib.gk_shared_prefix_list_build(*map(ptr, arrays), None if request is None else ptr(request), len(arrays[0]), ptr(prefix), len(prefix), *heads, window,
                                         ptr(words), capacity, ctypes.byref(lst))
    return rc, words, lst


def test_list_has_its_words():
    rc, _, lst = build(capacity=0)
    assert rc == capi.GK_ERR_WORKSPACE and lst.word_count > 0
    need = lst.word_count
    rc, words, lst = build(capacity=need)
    assert rc == capi.GK_OK and lst.rows == 2 and lst.word_count == need
    assert list(words[lst.map_at:lst.map_at + 2]) == [0, 1]
    assert list(words[lst.position_at:lst.position_at + 2]) == [700, 900]
    assert all(at % 4 == 0 for at in (lst.map_at, lst.position_at, lst.merges_at, lst.tiles_at, lst.workers_at,
                                      lst.segments_at))
    rc, words, _ = build(capacity=need + 5)
    assert rc == capi.GK_OK and (words[need:] == -7).all()


@pytest.mark.parametrize("change,message", [
    ({"size": 8}, "struct_size"), ({"heads": (32, 8, 96)}, "head geometry"), ({"heads": (30, 8, 128)}, "head geometry"),
    ({"heads": (129, 1, 128)}, "head geometry"), ({"group": (1, 0), "prefix": (64, 64)}, "order of their groups"),
    ({"group": (0, 1)}, "order of their groups"), ({"group": (-1, 0)}, "order of their groups"),
    ({"pos": (639, 900)}, "behind its group's prefix"), ({"rows": (0, 1)}, "behind its group's prefix"),
    ({"prefix": (-1,)}, "behind its group's prefix"), ({"pos": (700, 2**31 - 40)}, "behind its group's prefix"),
    ({"rows": (65000, 1000)}, "too many rows"), ({"first": (), "rows": (), "pos": (), "group": ()}, "runs or groups"),
    ({"prefix": ()}, "runs or groups"), ({"request": (0, -1)}, "negative request"),
])
def test_build_refuses(change, message):
    rc, words, _ = build(**change)
    assert rc == capi.GK_ERR_INVALID_ARGUMENT and message in capi.load().gk_last_error().decode()
    assert (words == -7).all()


def attention_args():
    p, lst = capi.PrefillParams(), capi.SharedPrefixList()
    fake = 1 << 20  # never dereferenced: every refused call returns before a launch
    p.query = p.pool = p.block_tables = p.out = fake
    p.q_row_stride = p.out_row_stride = 32 * 128
    p.slots, p.bt_stride, p.block_size = 4096, 32, 128
    p.q_heads, p.kv_heads, p.head_dim, p.scale = 32, 8, 128, 0.1
    p.sliding_window = -1
    _, _, lst = build()
    lst.words = lst.row_request = fake
    return p, lst


@pytest.mark.parametrize("change,code,message", [
    (lambda p, lst: setattr(p, "struct_size", 8), capi.GK_ERR_INVALID_ARGUMENT, "struct_size"),
    (lambda p, lst: setattr(lst, "struct_size", 8), capi.GK_ERR_INVALID_ARGUMENT, "struct_size"),
    (lambda p, lst: setattr(p, "head_dim", 96), capi.GK_ERR_UNSUPPORTED, "head dimension"),
    (lambda p, lst: setattr(p, "scale", 0.0), capi.GK_ERR_INVALID_ARGUMENT, "scale"),
    (lambda p, lst: setattr(p, "out", None), capi.GK_ERR_INVALID_ARGUMENT, "null pointer"),
    (lambda p, lst: setattr(p, "q_row_stride", 100), capi.GK_ERR_INVALID_ARGUMENT, "16-byte aligned"),
    (lambda p, lst: setattr(lst, "words", None), capi.GK_ERR_INVALID_ARGUMENT, "null or misaligned"),
    (lambda p, lst: setattr(lst, "words", (1 << 20) + 4), capi.GK_ERR_INVALID_ARGUMENT, "null or misaligned"),
    (lambda p, lst: setattr(lst, "row_request", None), capi.GK_ERR_INVALID_ARGUMENT, "null or misaligned"),
    (lambda p, lst: setattr(lst, "worker_groups", lst.worker_groups + 1), capi.GK_ERR_INVALID_ARGUMENT, "counts"),
    (lambda p, lst: None, capi.GK_ERR_WORKSPACE, "workspace too small"),
])
def test_attention_refuses(change, code, message):
    lib = capi.load()
    p, lst = attention_args()
    need = lib.gk_shared_prefix_workspace_bytes(ctypes.byref(p), ctypes.byref(lst))
    assert need == 8 * lst.part_cols * (128 + 2) * 4
    change(p, lst)
    short = need - 1 if code == capi.GK_ERR_WORKSPACE else need
    assert lib.gk_shared_prefix_attention(ctypes.byref(p), ctypes.byref(lst), ctypes.c_void_p(1 << 20), short,
                                          None) == code
    assert message in lib.gk_last_error().decode()


@pytest.mark.parametrize("field,value", [("q_heads", 64), ("kv_heads", 16), ("head_dim", 64), ("sliding_window", 100)])
def test_attention_refuses_another_geometry(field, value):
    p, lst = attention_args()
    setattr(p, field, value)
    p.q_row_stride = p.out_row_stride = 64 * 128
    assert capi.load().gk_shared_prefix_attention(ctypes.byref(p), ctypes.byref(lst), ctypes.c_void_p(1 << 20), 1 << 40,
                                                  None) == capi.GK_ERR_INVALID_ARGUMENT
    assert "built for other heads" in capi.load().gk_last_error().decode()
