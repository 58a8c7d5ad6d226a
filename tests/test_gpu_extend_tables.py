"""extend_block_tables on the GPU against the same step done request by request
on the host, whole numbers throughout; then a serving loop on its tables."""

import numpy as np
import pytest
import torch

import gaudirt_amd
from tests.serving_reference import same_bits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def extension():
    gaudirt_amd.load_extension()


class Step:
    """`seqs`: (cached, new, parent row or -1). Parents' rows come behind the batch's, filled with `parent_tokens`."""

    def __init__(self, seed, seqs, *, page=16, context=512, parents=(), parent_tokens=0, free=None, head=0, slots=None,
                 with_map=True, spare_rows=4):
        rng = np.random.default_rng(seed)
        self.page, self.context, self.seqs = page, context, seqs
        self.width = -(-context // page)
        self.requests = len(seqs) + len(parents) + spare_rows
        order = rng.permutation(self.requests)
        self.rows, parent_rows = order[:len(seqs)], order[len(seqs):len(seqs) + len(parents)]
        total = 1 + sum(-(-min(context, c + max(n, 0)) // page) for c, n, _ in seqs) + len(parents) * self.width + 8
        pages = rng.permutation(np.arange(1, total + 1))
        self.slots = (total + 1) * page if slots is None else slots
        self.tables = np.full((self.requests, self.width), -1, dtype=np.int32)
        at = 0
        fills = [(r, c) for r, (c, _, p) in zip(self.rows, seqs) if p < 0] + [(r, parent_tokens) for r in parent_rows]
        self.mapping = np.full((self.requests, context), -1, dtype=np.int32)
        for row, tokens in fills:
            tokens = min(max(tokens, 0), context)
            count = -(-tokens // page)
            self.tables[row, :count] = pages[at:at + count]
            at += count
            t = np.arange(tokens)
            self.mapping[row, :tokens] = self.tables[row, t // page] * page + t % page
        self.parents = np.array([parent_rows[p] if p >= 0 else -1 for _, _, p in seqs], dtype=np.int64)
        self.has_parents = len(parents) > 0
        self.free = np.concatenate([np.zeros(head, dtype=np.int64), pages[at:]]) if free is None else np.asarray(free)
        self.head = head
        self.with_map = with_map

    def expected(self, max_rows):
        """Outputs of the documented step on copies of the tables."""
        tables, mapping, page = self.tables.copy(), self.mapping.copy(), self.page
        room = min(self.width * page, self.context if self.with_map else 1 << 31)
        locations, requests, positions = [], [], []
        head, status, bad = self.head, 0, -1
        for s, ((c, n, _), row) in enumerate(zip(self.seqs, self.rows)):
            parent = int(self.parents[s])
            if not (0 <= row < self.requests and parent < self.requests):
                status, bad = 1, s
            elif c < 0 or n < 0 or c + n > room:
                status, bad = 2, s
            elif parent >= 0 and (c % page or parent == row):
                status, bad = 3, s
            elif len(locations) + n > max_rows:
                status, bad = 4, s
            else:
                held = -(-c // page)
                need = -(-(c + n) // page) - held
                if need > len(self.free) - head:
                    status, bad = 5, s
                else:
                    if parent >= 0:
                        tables[row, :held] = tables[parent, :held]
                        mapping[row, :c] = mapping[parent, :c]
                    for e in range(need):
                        p = int(self.free[head + e])
                        tables[row, held + e] = p if 0 <= p < self.slots // page else -1
                    head += need
                    for t in range(c, c + n):
                        p = int(tables[row, t // page])
                        mapping[row, t] = p * page + t % page if p >= 0 else -1
                        locations.append(mapping[row, t])
                        requests.append(row)
                        positions.append(t)
            if status:
                break
        if status:
            tables, mapping, head = self.tables, self.mapping, self.head
            locations, requests, positions = [], [], []
        rows = len(locations)
        pad = lambda v, fill: np.array(list(v) + [fill] * (max_rows - rows), dtype=np.int32)  # noqa: E731
        lens = np.array([c + (0 if status else n) for c, n, _ in self.seqs], dtype=np.int64)
        return (pad(locations, -1), pad(requests, 0), pad(positions, 0), lens,
                np.array([rows, head, status, bad], dtype=np.int32), tables, mapping if self.with_map else self.mapping)

    def check(self, max_rows=None, requests=torch.int32, lengths=torch.int64, pages=torch.int64, strided=False):
        if max_rows is None:
            max_rows = sum(n for _, n, _ in self.seqs)
        put = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to(device="cuda", dtype=t)  # noqa: E731

        def vector(a, t):
            v = put(a, t)
            return torch.stack([v, v - 7], 1)[:, 0] if strided else v

        tables, mapping = put(self.tables, torch.int32), put(self.mapping, torch.int32)
        got = torch.ops.gaudirt.extend_block_tables(
            tables, mapping if self.with_map else None, vector(self.rows, requests),
            vector([c for c, _, _ in self.seqs], lengths), vector([n for _, n, _ in self.seqs], lengths),
            vector(self.free, pages), put([self.head], torch.int32) if self.head else None,
            vector(self.parents, requests) if self.has_parents else None, self.page, self.slots, max_rows)
        names = ("locations", "row_requests", "positions", "seq_lens", "counts", "tables", "mapping")
        expected = self.expected(max_rows)
        for name, a, e in zip(names, (*got, tables, mapping), expected):
            assert np.array_equal(a.cpu().numpy(), e), name
        return expected


@pytest.mark.parametrize("page", [1, 2, 16, 64, 128])
@pytest.mark.parametrize("with_map", [True, False])
def test_steps(page, with_map):
    rng = np.random.default_rng(page)
    for n in (1, 2, 7, 64, 300):
        seqs = [(int(rng.integers(0, 400)), int(rng.integers(0, 100)), -1) for _ in range(n)]
        Step(n, seqs, page=page, with_map=with_map).check()
        Step(n, [(c, 1, -1) for c, _, _ in seqs], page=page, with_map=with_map).check()


@pytest.mark.parametrize("requests,lengths,pages", [(torch.int64, torch.int32, torch.int32),
                                                    (torch.int32, torch.int32, torch.int64),
                                                    (torch.int64, torch.int64, torch.int32)])
@pytest.mark.parametrize("strided", [False, True])
def test_types_and_strides(requests, lengths, pages, strided):
    seqs = [(32, 5, 0), (0, 40, -1), (64, 0, 0), (17, 3, -1)]
    Step(3, seqs, parents=(0,), parent_tokens=70).check(requests=requests, lengths=lengths, pages=pages, strided=strided)


@pytest.mark.parametrize("page", [1, 16, 128])
@pytest.mark.parametrize("with_map", [True, False])
def test_forks(page, with_map):
    whole = 256
    seqs = [(whole, 3, 0), (whole, 0, 0), (128, 9, 0), (0, 4, 0), (50, 60, -1)] + [(whole, i % 40, i % 2) for i in range(60)]
    Step(4, seqs, page=page, parents=(0, 1), parent_tokens=300, with_map=with_map).check()


def test_parent_extended_in_the_same_step():
    step = Step(5, [(48, 7, -1), (32, 4, 0), (48, 1, 0)], parents=(0,), parent_tokens=48)
    # The first sequence's row is the others' parent: they take the tokens that it held before.
    step.parents[1:] = step.rows[0]
    step.check()


def test_no_sequences_no_rows():
    Step(6, []).check()
    Step(7, [(16, 0, -1), (5, 0, -1)]).check(max_rows=0)
    Step(8, [(16, 0, -1), (5, 2, -1), (0, 0, -1)]).check(max_rows=9)


def test_rows_behind_the_last_are_no_tokens():
    expected = Step(9, [(30, 4, -1), (0, 17, -1)]).check(max_rows=5000)
    assert expected[4][0] == 21 and (expected[0][21:] == -1).all()


def test_many_sequences():
    rng = np.random.default_rng(10)
    for n in (1024, 1025, 8192):
        Step(n, [(int(c), int(k), -1) for c, k in zip(rng.integers(0, 60, n), rng.integers(0, 4, n))], page=4,
             context=64).check()


def test_long_prompts():
    Step(11, [(0, 32768, -1), (1, 20000, -1), (129, 7, -1)], page=128, context=32768).check()
    Step(12, [(0, 9999, -1), (16, 16, -1)], page=16, context=10000).check()


def test_free_list_head_and_bad_pages():
    Step(13, [(30, 20, -1), (0, 17, -1)], head=5).check()
    Step(14, [(0, 40, -1), (0, 17, -1)], free=[3, -1, 1 << 40, 5, 6, 7]).check()  # outside the pool: entered as -1
    Step(15, [(0, 40, -1)], free=[8, 9, 10], slots=9 * 16).check()                # page 8 is the last one


@pytest.mark.parametrize("seqs", [2, 1100])
@pytest.mark.parametrize("page", [-1, 1 << 20, (1 << 28) + 1])
def test_cached_pages_outside_the_pool(seqs, page):
    # A table row that was never filled: the tokens that continue such a page get no slot, whatever their page's entry is.
    put = lambda v, t=torch.int32: torch.tensor(v, device="cuda", dtype=t)  # noqa: E731
    tables = torch.full((seqs, 4), page, device="cuda", dtype=torch.int32)
    locations, requests, positions, lengths, counts = torch.ops.gaudirt.extend_block_tables(
        tables, None, put(list(range(seqs))), put([5] * seqs), put([3] + [0] * (seqs - 2) + [12]), put([1, 2], torch.int64),
        None, None, 16, 64, 15)
    assert counts.tolist() == [15, 1, 0, -1]
    assert locations.tolist() == [-1] * 14 + [16] and positions.tolist() == [5, 6, 7] + list(range(5, 17))
    assert tables[-1].tolist() == [page, 1, page, page]


@pytest.mark.parametrize("step,rows,status", [
    (dict(seqs=[(0, 3, -1), (500, 13, -1)]), None, 2), (dict(seqs=[(0, 3, -1), (513, 0, -1)]), None, 2),
    (dict(seqs=[(-1, 3, -1)]), None, 2), (dict(seqs=[(5, 1, -1), (5, -1, -1)]), 9, 2),
    (dict(seqs=[(17, 3, 0)], parents=(0,), parent_tokens=40), None, 3),
    (dict(seqs=[(0, 30, -1), (0, 30, -1)]), 59, 4), (dict(seqs=[(0, 30, -1), (0, 30, -1)], free=[1, 2, 3]), None, 5),
    (dict(seqs=[(16, 0, -1), (16, 1, -1)], free=[]), None, 5), (dict(seqs=[(1 << 30, 1 << 30, -1)]), 8, 2),
])
def test_status(step, rows, status):
    s = Step(16, step.pop("seqs"), **step)
    expected = s.check(max_rows=rows)
    assert expected[4][2] == status and expected[4][0] == 0


def test_status_of_rows_outside_the_tables():
    for which, bad in (("rows", -1), ("rows", 1 << 20), ("parents", 1 << 20)):
        s = Step(17, [(16, 3, -1), (16, 3, 0)], parents=(0,), parent_tokens=16)
        getattr(s, which)[1] = bad
        assert s.check()[4][2] == 1
    s = Step(18, [(16, 3, 0)], parents=(0,), parent_tokens=16)
    s.parents[0] = s.rows[0]
    assert s.check()[4][2] == 3


def test_captured_and_replayed():
    s = Step(19, [(0, 0, -1)] * 6, page=4, context=256)
    put = lambda a, t=torch.int64: torch.tensor(a, device="cuda", dtype=t)  # noqa: E731
    tables, mapping = (torch.from_numpy(a).cuda() for a in (s.tables, s.mapping))
    requests, lens, new = put(s.rows.tolist(), torch.int32), put([0] * 6), put([1, 2, 3, 0, 1, 5])
    free, head = put(list(range(1, 400))), put([0], torch.int32)
    step = lambda: torch.ops.gaudirt.extend_block_tables(tables, mapping, requests, lens, new, free, head, None, 4, 4096, 32)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
            lens.copy_(out[3])
            head.copy_(out[4][1:2])
        taken = 0
        for i in range(6):
            before = lens.tolist()
            graph.replay()
            side.synchronize()
            assert lens.tolist() == [b + n for b, n in zip(before, [1, 2, 3, 0, 1, 5])]
            taken += sum(-(-a // 4) - -(-b // 4) for a, b in zip(lens.tolist(), before))
            assert head.item() == taken and out[4].tolist() == [12, taken, 0, -1]
            for r, n in zip(s.rows.tolist(), lens.tolist()):
                t = torch.arange(n, device="cuda")
                assert torch.equal(mapping[r, :n], tables[r][t // 4] * 4 + t.int() % 4)
                assert (mapping[r, n:] == -1).all()
        held = tables[tables >= 0]
        assert len(held) == taken == len(held.unique())


def test_refusals():
    s = Step(20, [(0, 3, -1), (5, 1, -1)])
    put = lambda a, t=torch.int64: torch.tensor(a, device="cuda", dtype=t)  # noqa: E731
    base = dict(block_tables=torch.from_numpy(s.tables).cuda(), mapping=torch.from_numpy(s.mapping).cuda(),
                requests=put([0, 1]), prefixes=put([0, 5]), lengths=put([3, 1]), free_pages=put([1, 2, 3]), free_head=None,
                parents=None, page_size=16, slots=4096, max_rows=4)
    tables = base["block_tables"].clone()
    for change, message in [
            ({"block_tables": base["block_tables"].long()}, "int32 tables"), ({"block_tables": base["block_tables"].t()}, "int32 tables"),
            ({"mapping": base["mapping"][:3]}, "as many rows"), ({"mapping": base["mapping"].cpu()}, "as many rows"),
            ({"requests": put([0])}, "do not match"), ({"prefixes": put([0, 5], torch.int32)}, "do not match"),
            ({"lengths": put([[3, 1]])}, "vectors"), ({"requests": put([0.0, 1.0], torch.float32)}, "vectors"),
            ({"parents": put([-1, -1], torch.int32)}, "do not match"), ({"parents": put([-1])}, "do not match"),
            ({"free_head": put([0])}, "head"), ({"free_head": put([0, 0], torch.int32)}, "head"),
            ({"page_size": 24}, "page size"), ({"page_size": 0}, "page size"), ({"slots": 0}, "page size"),
            ({"max_rows": -1}, "page size"), ({"slots": 1 << 40}, "page size"),
            ({k: torch.zeros(8193, dtype=torch.int64, device="cuda") for k in ("requests", "prefixes", "lengths")}, "8192")]:
        with pytest.raises(RuntimeError, match=message):
            torch.ops.gaudirt.extend_block_tables(**{**base, **change})
    assert torch.equal(base["block_tables"], tables)


@pytest.mark.parametrize("op", ["shared_prefix_attn", "paged_attn_alibi", "paged_attn"])
def test_serving_loop(op):
    """One prompt, forked into eight continuations, decoded for three steps: tables made on the device, attention
    over the scheduler's metadata, every step against dense attention in 64 bits of the tokens so far."""
    heads, kv_heads, d, page, slots, prompt, forks = 8, 2, 128, 16, 4096, 160, 8
    scale = d ** -0.5
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    normal = lambda *s: torch.empty(s, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)  # noqa: E731
    pool = gaudirt_amd.allocate_paged_kv(1, slots, kv_heads, d)
    views = gaudirt_amd.kv_pool_views(pool, 0)
    tables = torch.full((12, 32), -1, dtype=torch.int32, device="cuda")
    mapping = torch.full((12, 512), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(slots // page - 1, generator=torch.Generator().manual_seed(2)).cuda() + 1
    head = torch.zeros(1, dtype=torch.int32, device="cuda")
    put = lambda a: torch.tensor(a, dtype=torch.int64, device="cuda")  # noqa: E731
    slopes = torch.exp2(-torch.arange(1.0, heads + 1, device="cuda"))
    history = {}  # row -> (keys, values) of its tokens

    def step(rows, prefixes, lengths, parents, groups):
        nonlocal head
        total = sum(lengths)
        locations, row_requests, positions, lens, counts = torch.ops.gaudirt.extend_block_tables(
            tables, mapping, put(rows), put(prefixes), put(lengths), free, head, put(parents), page, slots, total)
        head = counts[1:2]
        assert counts.tolist()[2:] == [0, -1] and lens.tolist() == [p + n for p, n in zip(prefixes, lengths)]
        meta = torch.classes.gaudirt.PagedMetadata.from_device(locations, put(rows), positions, mapping, prefixes,
                                                               lengths, slots)
        q, k, v = normal(total, heads * d), normal(total, kv_heads * d), normal(total, kv_heads * d)
        if op == "shared_prefix_attn":
            out = torch.ops.gaudirt.shared_prefix_attn(q, k, v, *views, meta, *groups, d, scale)
        elif op == "paged_attn_alibi":
            out = torch.ops.gaudirt.paged_attn_alibi(q, k, v, *views, meta, slopes, d, scale)
        else:
            out = torch.ops.gaudirt.paged_attn(q, k, v, *views, meta, d, scale)
        at = 0
        for row, prefix, n, parent in zip(rows, prefixes, lengths, parents):
            if parent >= 0:
                history[row] = history[parent]
            new = [x[at:at + n].view(n, kv_heads, d) for x in (k, v)]
            history[row] = [torch.cat([h[:prefix], x]) if row in history else x for h, x in zip(history.get(row, new), new)]
            keys, values = (x.double().repeat_interleave(heads // kv_heads, 1).transpose(0, 1).contiguous() for x in history[row])
            score = q[at:at + n].double().view(n, heads, d).transpose(0, 1).contiguous() @ keys.transpose(1, 2).contiguous() * scale
            distance = (torch.arange(prefix + n, device="cuda") - torch.arange(prefix, prefix + n, device="cuda")[:, None])
            if op == "paged_attn_alibi":
                score = score + slopes.double()[:, None, None] * distance
            weight = torch.softmax(score.masked_fill(distance > 0, -float("inf")), dim=2)
            exact = (weight @ values).transpose(0, 1).reshape(n, -1)
            size = (weight @ values.abs()).transpose(0, 1).reshape(n, -1)
            # Twice the rounding of the weights, the output's own, and 1e-3 of the weights' sum for fp32 scores.
            bound = 2.0 ** -8 * (2 * size + exact.abs()) * 1.02 + 1e-3 * size
            assert bool(((out[at:at + n].double() - exact).abs() <= bound).all())
            at += n

    step([3], [0], [prompt], [-1], ([prompt], [0]))
    rows = [0, 1, 2, 4, 5, 6, 7, 8]
    lens = [prompt] * forks
    for i in range(3):
        new = [1 + (r + i) % 3 for r in rows]
        step(rows, lens, new, [3 if i == 0 else -1] * forks, ([sum(new)], [prompt]))
        lens = [a + b for a, b in zip(lens, new)]
    assert same_bits(pool[:, :, :, :page], torch.zeros_like(pool[:, :, :, :page])), "page 0 was never handed out"
