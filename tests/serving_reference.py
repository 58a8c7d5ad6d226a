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

import math

import numpy as np
import torch

import gaudirt_amd


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
