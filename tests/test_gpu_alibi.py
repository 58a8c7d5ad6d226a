"""paged_attn_alibi on the GPU against 64-bit attention row by row (bounds in
tests/serving_reference.py), and what it refuses."""

import ctypes

import pytest
import torch

import gaudirt_amd
from gaudirt_amd import capi
from tests.serving_reference import Batch, same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def extension():
    gaudirt_amd.load_extension()


def slopes_of(b, kind="steep"):
    h = torch.arange(b.q_heads, device="cuda", dtype=torch.float32)
    return {"steep": torch.exp2(-8 * (h + 1) / b.q_heads), "flat": 1e-3 * (h + 1), "zero": 0 * h,
            "rising": -0.02 * (1 + h / b.q_heads), "mixed": 0.05 * (h % 3 - 1)}[kind]


def run(b, slopes, softcap=0.0, window=-1, **kw):
    return torch.ops.gaudirt.paged_attn_alibi(kw.get("query", b.query), b.key, b.value, *b.views,
                                              kw.get("metadata", b.metadata), slopes, b.d, b.scale, softcap, window)


def check(b, kind="steep", **how):
    slopes, pool = slopes_of(b, kind), b.stored()
    out = run(b, slopes, **how)
    b.check(out, slopes=slopes, **how)
    assert same_bits(b.pool, pool), "pool bytes differ"
    return out


def decode(lengths):
    return [(0, n, 1) for n in lengths]


HEADS = [(32, 8, 128), (8, 8, 128), (14, 2, 64), (16, 8, 256), (24, 8, 128), (16, 8, 128), (32, 1, 128), (40, 2, 64)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [1, 4, 16, 128])
def test_decode_short(heads, page):
    check(Batch(1, decode([0, 1, 30, 31, 32, 63, 200, 511]), [0], heads=heads, page=page))


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [1, 16, 128])
def test_decode_long(heads, page):
    # Too long for one workgroup a unit: the balanced schedule with its merge.
    check(Batch(2, decode([0, 5000, 4097, 64, 2999]), [0], heads=heads, page=page), kind="flat")


@pytest.mark.parametrize("heads", HEADS)
def test_batch_invariant_partitions(heads):
    b = Batch(3, decode([0, 5000, 4097, 64, 2999]) + [(0, 100, 40)], [0], heads=heads)
    gaudirt_amd.set_batch_invariant_decode(True, 1024)
    try:
        check(b, kind="flat")
    finally:
        gaudirt_amd.set_batch_invariant_decode(False)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [1, 8, 128])
def test_prefill(heads, page):
    check(Batch(4, [(0, 0, 100), (0, 37, 8), (0, 300, 65), (0, 5, 3)], [0], heads=heads, page=page))


def test_prefill_cut_along_its_keys():
    check(Batch(5, [(0, 5000, 150)], [0], heads=(8, 2, 128)), kind="flat")
    check(Batch(6, [(0, 3840, 120)], [0], heads=(14, 2, 64), page=1), kind="flat")


@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (16, 8, 256), (8, 8, 128)])
@pytest.mark.parametrize("how", [{"softcap": 30.0}, {"window": 33}, {"softcap": 50.0, "window": 500}, {"window": 1}])
@pytest.mark.parametrize("kind", ["steep", "rising", "mixed"])
def test_softcap_window_and_slopes(heads, how, kind):
    check(Batch(7, decode([0, 3, 100, 700, 4500]) + [(0, 400, 70)], [0], heads=heads), kind=kind, **how)


def test_zero_slopes_are_paged_attn():
    b = Batch(8, decode([0, 3, 100, 700]) + [(0, 400, 70)], [0])
    out = check(b, kind="zero")
    plain = torch.ops.gaudirt.paged_attn(*b.inputs(), b.d, b.scale)
    assert float((out.float() - plain.float()).abs().max()) < 0.02


def test_slope_that_hides_all_but_the_nearest():
    # 2^-1e30 beyond the own key: its value alone, exactly.
    b = Batch(9, decode([0, 3, 100, 6000]) + [(0, 40, 33)], [0], heads=(8, 8, 128))
    out = run(b, torch.full([b.q_heads], 1e30, device="cuda"))
    assert same_bits(out, b.value)


@pytest.mark.parametrize("kind", ["device", "scheduler"])
def test_device_metadata(kind):
    check(Batch(10, decode([0, 3, 100, 700, 5000]) + [(0, 400, 70)], [0], metadata=kind))


def test_strided_slopes_and_query():
    b = Batch(11, decode([0, 3, 100, 700]), [0])
    slopes = slopes_of(b)
    expected = run(b, slopes)
    assert same_bits(run(b, torch.stack([slopes, 0 * slopes], 1)[:, 0]), expected)
    wide = torch.zeros(b.rows, b.query.shape[1] + 8, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:-5] = b.query
    assert same_bits(run(b, slopes, query=wide[:, 3:-5]), expected)


def test_captured_and_replayed():
    b = Batch(12, decode([0, 3, 100, 700, 5000]) + [(0, 2000, 70)], [0])
    slopes = slopes_of(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        metadata = b.make_metadata()
        run(b, slopes, metadata=metadata)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run(b, slopes, metadata=metadata)
        for i in range(4):
            b.query.normal_()
            slopes.mul_(0.7)
            graph.replay()
            side.synchronize()
            b.check(out, slopes=slopes)
            assert same_bits(run(b, slopes, metadata=metadata), out)
            side.synchronize()


def test_refusals():
    b = Batch(13, decode([0, 3, 100]), [0])
    pool, good = b.pool.clone(), slopes_of(b)
    for bad in (good[:-1], good.double(), good.cpu(), good[None], good.bfloat16()):
        with pytest.raises(RuntimeError, match="slopes"):
            run(b, bad)
    with pytest.raises(RuntimeError, match="scale"):
        run(b, good, softcap=-1.0)
    with pytest.raises(RuntimeError, match="sliding window|scale"):
        run(b, good, window=0)
    assert same_bits(b.pool, pool)


def test_c_entries_refuse_null_slopes():
    lib, p = capi.load(), capi.DecodeParams()
    p.rows = 1
    assert lib.gk_paged_decode_alibi(ctypes.byref(p), None, None, 0, None) == capi.GK_ERR_INVALID_ARGUMENT
    assert "slopes" in lib.gk_last_error().decode()
    f, lst = capi.PrefillParams(), capi.PrefillList()
    assert lib.gk_paged_prefill_alibi(ctypes.byref(f), ctypes.byref(lst), None, None, 0,
                                      None) == capi.GK_ERR_INVALID_ARGUMENT
    assert "slopes" in lib.gk_last_error().decode()
