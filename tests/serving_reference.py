"""A batch of requests in a paged pool and its attention in 64 bits, for the
tests of shared_prefix_attn and paged_attn_alibi.

The bound on a kernel's output. Probabilities are rounded to bf16 before they
meet V (half a step: 2^-8 of each), the sum that divides may be that of the
rounded ones, and the output is rounded once more, so with A = sum_t w_t |v_t|
and w the softmax weights

    |out - o| <= 2^-8 (2 A + |o|) (1 + 2^-6) + w-error,

where the last factor covers products of roundings. Scores are fp32 sums of d
products of bf16 values: off by at most (d + 3) 2^-24 S, S = max_t sum_i |q_i
k_i| scale, plus 2^-18 for a softcap's exponential and reciprocal times the cap
and 2^-23 of a bias; a weight is off by e times that, twice for the sum. Every
term is computed from the case itself.
"""

import ctypes
import math

import numpy as np
import torch

import gaudirt_amd
from gaudirt_amd import capi


class Batch:
    """Requests (group, shared tokens, own cached tokens, new tokens), a group's side by side, on pages of `page`
    tokens in scattered order. Slots that hold no token are NaN."""

    def __init__(self, seed, requests, prefix, *, heads=(32, 8, 128), page=16, metadata="host", spare=3, value_scale=1.0):
        rng = np.random.default_rng(seed)
        self.q_heads, self.kv_heads, self.d = heads
        self.requests, self.prefix, self.page = requests, prefix, page
        shared = [p // page for p in prefix]
        starts = [prefix[g] + own for g, own, _ in requests]
        ends = [s + n for s, (_, _, n) in zip(starts, requests)]
        total = sum(shared) + sum(-(-e // page) - shared[g] for e, (g, _, _) in zip(ends, requests))
        blocks = rng.permutation(total + spare)
        context = max(ends)
        mapping = np.full((len(requests), context), -1, dtype=np.int32)
        at, head = 0, {}
        for r, (g, _, _) in enumerate(requests):
            if g not in head:
                head[g] = blocks[at:at + shared[g]]
                at += shared[g]
            mine = -(-ends[r] // page) - shared[g]
            table = np.concatenate([head[g], blocks[at:at + mine]])
            at += mine
            t = np.arange(ends[r])
            mapping[r, :ends[r]] = table[t // page] * page + t % page
        self.mapping, self.slots = mapping, len(blocks) * page
        news = [n for _, _, n in requests]
        self.row_request = np.repeat(np.arange(len(requests)), news)
        self.positions = np.concatenate([np.arange(s, s + n) for s, n in zip(starts, news)])
        self.locations = mapping[self.row_request, self.positions].astype(np.int64)
        self.rows = len(self.positions)
        self.group_prefix = [s * page for s in shared]  # what whole pages share
        self.group_rows = [sum(n for g, _, n in requests if g == k) for k in range(len(prefix))]
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)

        def normal(*shape):
            return torch.empty(shape, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)

        self.pool = gaudirt_amd.allocate_paged_kv(1, self.slots, self.kv_heads, self.d)
        self.pool.normal_(generator=gen)
        self.pool[:, 1] *= value_scale
        held = np.zeros(self.slots, dtype=bool)
        held[mapping[mapping >= 0]] = True
        self.pool[0][:, :, torch.from_numpy(~held).cuda()] = float("nan")
        self.query = normal(self.rows, self.q_heads * self.d)
        self.key, self.value = normal(self.rows, self.kv_heads * self.d), normal(self.rows, self.kv_heads * self.d)
        self.scale = float(np.float32(1 / math.sqrt(self.d)))
        self.metadata = self.make_metadata(metadata)
        self.views = gaudirt_amd.kv_pool_views(self.pool, 0)

    def make_metadata(self, kind="host"):
        cls = torch.classes.gaudirt.PagedMetadata
        if kind == "host":
            return cls(torch.from_numpy(self.locations), torch.from_numpy(self.row_request),
                       torch.from_numpy(self.positions), torch.from_numpy(self.mapping), self.slots)
        cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        lengths = [n for _, _, n in self.requests]
        prefixes = [self.prefix[g] + own for g, own, _ in self.requests]
        args = (cuda(self.locations), torch.arange(len(lengths), device="cuda"), cuda(self.positions),
                cuda(self.mapping), prefixes, lengths, self.slots)
        return cls.from_device(*args) if kind == "device" else cls._from_scheduler(*args, None, 0)

    def inputs(self):
        return self.query, self.key, self.value, *self.views, self.metadata

    def stored(self):
        """The pool after the new rows' store."""
        pool = self.pool.clone()
        where = torch.from_numpy(self.locations).cuda()
        for i, new in enumerate((self.key, self.value)):
            pool[0, i][:, where] = new.view(self.rows, self.kv_heads, self.d).transpose(0, 1)
        return pool

    def attend(self, *, softcap=0.0, window=-1, slopes=None):
        """(outputs, bounds) in 64 bits."""
        pool, d, group = self.stored()[0], self.d, self.q_heads // self.kv_heads
        out = torch.zeros(self.rows, self.q_heads, d, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        query = self.query.double().view(self.rows, self.q_heads, d)
        row = 0
        for r, (g, own, n) in enumerate(self.requests):
            start = self.prefix[g] + own
            where = torch.from_numpy(self.mapping[r, :start + n]).cuda().long()
            at = torch.arange(start + n, device="cuda")
            position = torch.arange(start, start + n, device="cuda")[:, None]
            seen = at <= position
            if window > 0:
                seen &= at > position - window
            for h in range(self.q_heads):
                k, v = pool[0, h // group][where].double(), pool[1, h // group][where].double()
                q = query[row:row + n, h]
                size = float((q.abs() @ k.abs().t()).masked_fill(~seen, 0).max()) * self.scale
                score = q @ k.t() * self.scale
                error = (d + 3) * 2.0 ** -24 * size + 2.0 ** -22 * score.abs()
                if softcap > 0:
                    score = softcap * torch.tanh(score / softcap)
                    error += softcap * 2.0 ** -18
                if slopes is not None:
                    bias = slopes[h].double() * (at - position).double()
                    error = error + 3 * 2.0 ** -23 * (bias.abs() + score.abs())
                    score = score + bias
                weight = torch.softmax(score.masked_fill(~seen, -math.inf), dim=1)
                v = torch.where(seen.any(0)[:, None], v, torch.zeros_like(v))
                o = weight @ v
                a = weight @ v.abs()
                w_error = 2 * math.e * ((weight * error) @ v.abs() + (weight * error).sum(1, keepdim=True) * a)
                out[row:row + n, h] = o
                bound[row:row + n, h] = 2.0 ** -8 * (2 * a + o.abs()) * (1 + 2.0 ** -6) + w_error
            row += n
        return out.view(self.rows, -1), bound.view(self.rows, -1)

    def check(self, actual, **kind):
        expected, bound = self.attend(**kind)
        assert actual.shape == expected.shape and actual.dtype == torch.bfloat16
        assert torch.isfinite(actual).all(), "an output is not finite"
        excess = (actual.double() - expected).abs() / bound
        assert float(excess.max()) <= 1.0, f"{float(excess.max()):.3f} times the bound at {int(excess.argmax())}"


def same_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def shared_prefix_c(b, softcap=0.0, window=-1, ride_along=False, known_requests=True, page=None):
    """The batch through gk_shared_prefix_list_build and gk_shared_prefix_attention, whatever its size (the operator
    lets short batches attend row by row): the new rows stored by gk_kv_store first, or with ride_along by the call
    itself. Rows of the output that the call does not write are NaN."""
    lib, page = capi.load(), page or b.page
    as_i32 = lambda a: np.ascontiguousarray(a, dtype=np.int32)  # noqa: E731
    news = as_i32([n for _, _, n in b.requests])
    first = as_i32(np.concatenate([[0], np.cumsum(news)[:-1]]))
    pos = as_i32([b.prefix[g] + own for g, own, _ in b.requests])
    group, prefix = as_i32([g for g, _, _ in b.requests]), as_i32(b.group_prefix)
    request = as_i32(np.arange(len(news)))
    host = lambda a: ctypes.c_void_p(a.ctypes.data)  # noqa: E731
    words, lst = np.zeros(1 << 20, dtype=np.int32), capi.SharedPrefixList()
    capi.check(lib.gk_shared_prefix_list_build(host(first), host(news), host(pos), host(group), host(request) if known_requests else None,
                                               len(news), host(prefix),
                                               len(prefix), b.q_heads, b.kv_heads, b.d, window, host(words), words.size,
                                               ctypes.byref(lst)))
    device_words = torch.from_numpy(words[:lst.word_count].copy()).cuda()
    row_request = torch.from_numpy(as_i32(b.row_request)).cuda()
    tables = b.mapping[:, ::page].copy()
    tables[tables >= 0] //= page
    tables = torch.from_numpy(tables).cuda()
    locations = torch.from_numpy(as_i32(b.locations)).cuda()
    out = torch.full((b.rows, b.q_heads * b.d), float("nan"), dtype=torch.bfloat16, device="cuda")
    lst.words, lst.row_request = device_words.data_ptr(), row_request.data_ptr()
    if ride_along:
        assert lst.can_store
        lst.new_key, lst.new_value, lst.new_kv_row_stride = b.key.data_ptr(), b.value.data_ptr(), b.key.stride(0)
    else:
        capi.check(lib.gk_kv_store(capi.ptr(b.key), capi.ptr(b.value), b.key.stride(0), b.value.stride(0),
                                   capi.ptr(locations), b.rows, capi.ptr(b.pool), b.slots, b.kv_heads, b.d,
                                   capi.current_stream()))
    p = capi.PrefillParams()
    p.query, p.q_row_stride = b.query.data_ptr(), b.query.stride(0)
    p.pool, p.slots = b.pool.data_ptr(), b.slots
    p.block_tables, p.bt_stride, p.block_size = tables.data_ptr(), tables.stride(0), page
    p.q_heads, p.kv_heads, p.head_dim = b.q_heads, b.kv_heads, b.d
    p.scale, p.softcap, p.sliding_window = b.scale, softcap, window
    p.out, p.out_row_stride = out.data_ptr(), out.stride(0)
    need = lib.gk_shared_prefix_workspace_bytes(ctypes.byref(p), ctypes.byref(lst))
    workspace = torch.full((need // 4 + 64,), float("nan"), device="cuda")  # a word past `need` must stay as it is
    capi.check(lib.gk_shared_prefix_attention(ctypes.byref(p), ctypes.byref(lst), capi.ptr(workspace), need,
                                              capi.current_stream()))
    assert torch.isnan(workspace[need // 4:]).all(), "the workspace was left"
    return out, bool(lst.can_store)
