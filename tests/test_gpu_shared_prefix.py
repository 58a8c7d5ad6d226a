"""shared_prefix_attn on the GPU against 64-bit attention row by row (bounds in
tests/serving_reference.py), and what it refuses."""

import numpy as np
import pytest
import torch

import gaudirt_amd
from tests.serving_reference import Batch, same_bits, shared_prefix_c

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def extension():
    gaudirt_amd.load_extension()


def run(b, group_rows=None, group_prefix=None, softcap=0.0, window=-1, **kw):
    return torch.ops.gaudirt.shared_prefix_attn(
        kw.get("query", b.query), b.key, b.value, *b.views, kw.get("metadata", b.metadata),
        b.group_rows if group_rows is None else group_rows, b.group_prefix if group_prefix is None else group_prefix,
        b.d, b.scale, softcap, window)


def check(b, **kind):
    """The operator, and the C entry with the new rows stored first and along the way: the operator lets short
    batches attend row by row."""
    before, expected_pool = b.pool.clone(), b.stored()
    out = run(b, **kind)
    b.check(out, **kind)
    assert same_bits(b.pool, expected_pool), "pool bytes differ"
    if b.q_heads // b.kv_heads <= 128:
        b.pool.copy_(before)
        stored, can_store = shared_prefix_c(b, **kind)
        b.check(stored, **kind)
        assert same_bits(b.pool, expected_pool)
        assert same_bits(shared_prefix_c(b, known_requests=False, **kind)[0], stored)
        if can_store:
            b.pool.copy_(before)
            along, _ = shared_prefix_c(b, ride_along=True, **kind)
            assert same_bits(along, stored) and same_bits(b.pool, expected_pool), "rows stored along the way"
    return out


def decode(groups, rows, own, step=37):
    """`rows` requests a group, own tokens 0, step, 2 step, ... modulo `own`."""
    return [(g, (i * step) % own, 1) for g in range(groups) for i in range(rows)]


HEADS = [(32, 8, 128), (8, 8, 128), (14, 2, 64), (16, 8, 256), (24, 8, 128), (64, 8, 128), (32, 1, 128), (48, 1, 64),
         (6, 3, 64), (40, 2, 256)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("page", [1, 16, 128])
def test_decode_rows(heads, page):
    check(Batch(1, decode(2, 9, 300), [513, 200], heads=heads, page=page))


@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (16, 8, 256)])
@pytest.mark.parametrize("kind", [{"softcap": 30.0}, {"window": 100}, {"softcap": 50.0, "window": 700}, {"window": 1}])
def test_softcap_and_window(heads, kind):
    # Windows that end inside the own tokens, inside the prefix, and at the row itself.
    check(Batch(2, decode(2, 12, 400), [513, 640], heads=heads), **kind)


@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (16, 8, 256), (8, 8, 128), (32, 1, 128)])
@pytest.mark.parametrize("new", [2, 3, 4, 7, 8, 15, 33])
def test_runs_of_new_tokens(heads, new):
    check(Batch(3, [(0, 5, new), (0, 0, 1), (0, 130, new + 1), (1, 7, new)], [300, 64], heads=heads))


@pytest.mark.parametrize("heads", [(32, 8, 128), (14, 2, 64), (16, 8, 256)])
def test_chunks_that_fill_a_tile(heads):
    # Runs of a tile's rows and more go to the prefill kernel, alone or beside others.
    check(Batch(4, [(0, 5, 200), (0, 17, 1), (1, 0, 300), (1, 3, 4)], [200, 96], heads=heads))
    check(Batch(5, [(0, 5, 150), (0, 17, 180)], [200], heads=heads))


@pytest.mark.parametrize("rows,prefix,own", [(1, 512, 1), (1, 16, 900), (2, 16, 1), (64, 1024, 40), (130, 48, 3),
                                             (300, 272, 60)])
def test_group_sizes(rows, prefix, own):
    check(Batch(6, decode(1, rows, own), [prefix], heads=(8, 2, 128)))


def test_no_shared_tokens():
    b = Batch(7, decode(3, 4, 200), [0, 64, 0])
    check(b)
    b = Batch(8, [(0, 0, 1), (0, 0, 1), (1, 0, 3)], [0, 5], page=16)  # first tokens: one key, own ones only
    assert b.group_prefix == [0, 0]
    check(b)


def test_declared_shorter_than_shared():
    b = Batch(9, decode(2, 8, 100), [640, 320])
    for prefix in ([0, 0], [1, 319], [33, 64], [640, 320]):
        b.check(run(b, group_prefix=prefix))
        b.group_prefix = prefix
        check(b)


def test_long_batches_share_through_the_operator():
    # Contexts beyond the one-launch decode kernel's: shared whatever the bytes; host and device metadata.
    for kind in ("host", "device", "scheduler"):
        b = Batch(30, decode(1, 20, 300) + [(1, 4, 5), (1, 9, 1)], [4000, 2600], metadata=kind)
        out = check(b)
        assert same_bits(out, shared_prefix_c(b)[0])


def test_rows_of_one_request_in_two_runs():
    # One request's chunk in two groups: the second part's rows see the first part's new keys.
    b = Batch(31, [(0, 5, 6), (0, 9, 1), (0, 11, 1)], [2400], heads=(8, 2, 128))
    expected, bound = b.attend()
    out = run(b, group_rows=[4, 4], group_prefix=[b.group_prefix[0], 16])
    assert bool(((out.double() - expected).abs() <= bound).all())
    assert same_bits(b.pool, b.stored())
    # The same rows, the request's later part first.
    order = [4, 5, 0, 1, 2, 3, 6, 7]
    for name in ("query", "key", "value"):
        setattr(b, name, getattr(b, name)[order].contiguous())
    b.locations, b.row_request, b.positions = b.locations[order], b.row_request[order], b.positions[order]
    b.pool.normal_()
    b.metadata = b.make_metadata()
    pool, sequential = b.stored(), []
    out = run(b, group_rows=[8], group_prefix=[b.group_prefix[0]])
    assert same_bits(b.pool, pool)
    for row in range(8):  # each row against plain attention over the stored pool
        n, group = int(b.positions[row]) + 1, b.q_heads // b.kv_heads
        at = torch.from_numpy(b.mapping[b.row_request[row], :n]).cuda().long()
        for h in range(b.q_heads):
            q = b.query[row].view(b.q_heads, b.d)[h].double()
            weight = torch.softmax(pool[0, 0, h // group][at].double() @ q * b.scale, 0)
            value = pool[0, 1, h // group][at].double()
            limit = 2.0 ** -8 * (2 * (weight @ value.abs()) + (weight @ value).abs()) * 1.02 + 1e-3 * (weight @ value.abs())
            sequential.append(bool(((out[row].view(b.q_heads, b.d)[h].double() - weight @ value).abs() <= limit).all()))
    assert all(sequential)


def test_many_groups():
    check(Batch(10, [(g, 3 * g % 50, 1 + g % 3) for g in range(70)], [16 * (g % 9) for g in range(70)]))


@pytest.mark.parametrize("kind", ["device", "scheduler"])
@pytest.mark.parametrize("page", [1, 16])
def test_device_metadata(kind, page):
    check(Batch(11, decode(2, 10, 300) + [(1, 4, 5)], [513, 200], page=page, metadata=kind))
    check(Batch(12, decode(1, 10, 300) + [(0, 4, 90)], [512], page=page, metadata=kind), window=400)


def test_long_prefix():
    check(Batch(13, decode(1, 40, 500), [20000], heads=(8, 2, 128), page=128))
    check(Batch(14, decode(1, 5, 500), [20000], heads=(14, 2, 64)))


# Groups of few columns, (rows of a group) x (heads a kv head), on prefixes of more than 512, or 1024, keys a CU of a kv
# head: all in tiles below, in waves of their own above, those of more than a quarter of a wave's columns between.
@pytest.mark.parametrize("heads,groups,rows,prefix", [
    ((32, 32, 64), 6, 3, 1600), ((32, 32, 64), 6, 20, 1600), ((64, 32, 64), 6, 16, 1600), ((64, 16, 128), 6, 4, 3001),
    ((64, 16, 128), 6, 7, 3001), ((32, 16, 256), 6, 1, 3001), ((32, 16, 256), 6, 8, 3001),
    ((32, 32, 64), 4, 5, 1600), ((64, 16, 128), 4, 3, 2600), ((32, 16, 256), 4, 5, 2600),
])
def test_few_columns_on_many_keys(heads, groups, rows, prefix):
    b = Batch(20, decode(groups, rows, 60), [prefix - 16 * g for g in range(groups)], heads=heads)
    check(b)
    check(b, softcap=30.0, window=1500)
    check(b, window=prefix - 40)


def test_extreme_values():
    # Scores of a few thousand, values near bf16's largest: weights of 0 and 1, no infinity on the way.
    b = Batch(15, decode(2, 9, 200), [300, 128], value_scale=1e37)
    b.query *= 300.0
    b.value *= 1e37
    exact, _ = b.attend()
    for out in (run(b), shared_prefix_c(b)[0]):
        assert torch.isfinite(out).all()
        assert float(((out.double() - exact).abs() / exact.abs().max()).max()) < 2.0 ** -6


def test_other_rows_infinities_stay_theirs():
    b = Batch(16, decode(1, 6, 80), [160], heads=(8, 2, 128))
    exact, _ = b.attend()
    b.key[2], b.value[2] = float("nan"), float("inf")
    others = [i for i in range(b.rows) if i != 2]
    for out in (run(b), shared_prefix_c(b)[0], shared_prefix_c(b, ride_along=True)[0]):
        assert torch.isfinite(out[others]).all() and not torch.isfinite(out[2]).all()
        assert float((out.double() - exact)[others].abs().max()) < 0.05


def test_batch_invariant_mode_attends_row_by_row():
    b = Batch(17, decode(2, 9, 300), [2513, 200])
    gaudirt_amd.set_batch_invariant_decode(True)
    try:
        out = run(b)
        plain = torch.ops.gaudirt.paged_attn(*b.inputs(), b.d, b.scale)
    finally:
        gaudirt_amd.set_batch_invariant_decode(False)
    assert same_bits(out, plain)
    b.check(out)


def test_repeats_and_layers_give_the_same_bits():
    b = Batch(18, decode(2, 20, 300) + [(1, 3, 9)], [513, 2800])
    first = run(b)
    second = Batch(19, decode(1, 30, 100), [2640])
    for _ in range(5):
        run(second)
        assert same_bits(run(b), first)
    assert same_bits(run(b, metadata=b.make_metadata()), first)


def test_strided_and_misaligned_inputs():
    b = Batch(20, decode(2, 9, 300), [2513, 200])
    expected = run(b)
    wide = torch.zeros(b.rows, b.query.shape[1] + 24, dtype=torch.bfloat16, device="cuda")
    for offset in (0, 8, 3):
        view = wide[:, offset:offset + b.query.shape[1]]
        view.copy_(b.query)
        assert same_bits(run(b, query=view), expected)
    turned = b.query.t().contiguous().t()
    assert same_bits(run(b, query=turned), expected)


def test_another_stream():
    b = Batch(21, decode(2, 9, 300), [2513, 200])
    expected = run(b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        metadata = b.make_metadata()
        out = run(b, metadata=metadata)
    side.synchronize()
    assert same_bits(out, expected)
    with pytest.raises(RuntimeError, match="stream"):
        run(b, metadata=metadata)


def test_two_streams_at_once():
    batches = [Batch(22 + i, decode(2, 20, 400), [2048, 2400]) for i in range(2)]
    expected = [run(b) for b in batches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    metadata = []
    for s, b in zip(streams, batches):
        with torch.cuda.stream(s):
            metadata.append(b.make_metadata())
            run(b, metadata=metadata[-1])
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (s, b) in enumerate(zip(streams, batches)):
            with torch.cuda.stream(s):
                outs[i].append(run(b, metadata=metadata[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(same_bits(o, expected[i]) for o in outs[i])


def test_captured_and_replayed():
    b = Batch(24, decode(2, 12, 300), [513, 2800])
    other = Batch(25, decode(1, 20, 100) + [(0, 3, 40)], [2640])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.metadata, other.metadata = b.make_metadata(), other.make_metadata()
        run(b)
        run(other)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run(b)
        second = torch.cuda.CUDAGraph()
        with torch.cuda.graph(second, stream=side):
            out2 = run(other)
        for i in range(4):
            for batch in (b, other):
                batch.query.normal_()
                batch.key.normal_()
                batch.value.normal_()
            graph.replay()
            second.replay()
            side.synchronize()
            b.check(out)
            other.check(out2)
            assert same_bits(run(b), out) and same_bits(run(other), out2)
            side.synchronize()
    torch.cuda.synchronize()


def test_first_call_is_not_captured():
    b = Batch(32, decode(1, 20, 100), [2640])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.metadata = b.make_metadata()
        torch.ops.gaudirt.paged_attn(*b.inputs(), b.d, b.scale)  # the attention plan itself is there
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="cannot be captured"):
            with torch.cuda.graph(graph, stream=side):
                run(b)
        check(b)
    torch.cuda.synchronize()


def test_page_aligned_prefixes_that_differ_in_one_page():
    b = Batch(33, decode(1, 9, 60), [2560], page=128)
    for page in (0, 7, 19):
        mapping = b.mapping.copy()
        other = np.setdiff1d(np.arange(b.slots // 128), mapping[mapping >= 0] // 128)[0]
        mapping[4, page * 128:(page + 1) * 128] = other * 128 + np.arange(128)
        metadata = torch.classes.gaudirt.PagedMetadata(
            torch.from_numpy(b.locations), torch.from_numpy(b.row_request), torch.from_numpy(b.positions),
            torch.from_numpy(mapping), b.slots)
        with pytest.raises(RuntimeError, match="do not share"):
            run(b, metadata=metadata)
        out = run(b, metadata=metadata, group_prefix=[page * 128])  # shared up to there
        assert torch.isfinite(out[[i for i in range(9) if i != 4]]).all()


def test_pool_beyond_32_bit_offsets():
    # Eight heads' K of 2^20 slots are 2 GiB; the last heads' rows lie past 2^32 bytes.
    b = Batch(26, decode(1, 6, 70), [160], heads=(16, 8, 256), page=16, spare=1 << 16)
    assert b.pool.numel() * 2 > 1 << 32
    check(b)


@pytest.mark.parametrize("change,message", [
    ({"group_rows": [9]}, "one row count"), ({"group_rows": [], "group_prefix": []}, "one row count"),
    ({"group_rows": [9, 8]}, "cover"), ({"group_rows": [9, 10]}, "out of range"), ({"group_rows": [18, 0]}, "out of range"),
    ({"group_prefix": [-1, 0]}, "out of range"), ({"group_prefix": [1 << 40, 0]}, "out of range"),
    ({"group_prefix": [514, 0]}, "inside its group's prefix"), ({"group_rows": [10, 8]}, "inside its group's prefix"),
    ({"group_rows": [10, 8], "group_prefix": [192, 192]}, "do not share"),
    ({"group_rows": [18], "group_prefix": [100]}, "do not share"), ({"window": 0}, "sliding window|scale, stream"),
    ({"softcap": -1.0}, "scale"), ({"softcap": float("nan")}, "scale"),
])
def test_refusals(change, message):
    b = Batch(27, decode(2, 9, 300), [513, 200])
    pool = b.pool.clone()
    with pytest.raises(RuntimeError, match=message):
        run(b, **change)
    assert same_bits(b.pool, pool), "a refused call wrote to the pool"


def test_refuses_wrong_tensors():
    b = Batch(28, decode(1, 4, 30), [64])
    call = lambda *a: torch.ops.gaudirt.shared_prefix_attn(*a, b.group_rows, b.group_prefix, b.d, b.scale)  # noqa: E731
    q, k, v, kp, vp, m = b.inputs()
    for args, message in [((q.float(), k, v, kp, vp, m), "BF16"), ((q[:3], k[:3], v[:3], kp, vp, m), "matching rows"),
                          ((q, k[:, :64], v, kp, vp, m), "do not match"), ((q, k, v, vp, kp, m), "combined storage"),
                          ((q, k, v, kp.contiguous(), vp, m), "head-major")]:
        with pytest.raises(RuntimeError, match=message):
            call(*args)


def test_more_than_128_heads_a_kv_head():
    b = Batch(29, decode(1, 5, 90), [160], heads=(160, 1, 64))
    out = check(b)
    assert same_bits(out, torch.ops.gaudirt.paged_attn(*b.inputs(), b.d, b.scale))
    assert np.isfinite(out.float().cpu().numpy()).all()
