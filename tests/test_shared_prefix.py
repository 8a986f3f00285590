"""Decode attention over shared prefixes (rh_shared_prefix_attention) against attention in 64 bits
over each token's whole context, and its refusals (on the CPU).

Tolerance, per output value: the result's rounding to fp16 (2^-11 of it, 2^-25 where it is
subnormal); the weights' rounding to fp16, 2^-11 of each, or 2^-25 absolute below 2^-14 (the greatest weight
of a slice is 1): 2^-11 sum w|v| + keys * 2^-25 * max|v|; scores summed in fp32: each is off by at
most (D + 2) * 2^-24 * scale * sum|q k|, which moves weights and their sum by that share each; and the
fp32 sums of the softmax and the joins, 64 roundings of 2^-24 on sum w|v| at most (a slice of n keys is
summed in n / 256 steps of 16 values and joined over 3 + 2 levels).
"""
import math

import numpy as np
import pytest

from helpers import bits_to_f32, f16_bits
from relay_amd import _lib


class Case:
    """Groups [(members, shared keys)] and per token (own keys); members 0 and shared 0: tokens on their own."""

    def __init__(self, groups, own, heads, kv_heads, D, bs=16, seed=0, spread=1.0, idle=(), ctx=None):
        rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.D, self.bs = heads, kv_heads, D, bs
        self.n = sum(m for m, _ in groups)
        own = [own[i % len(own)] for i in range(self.n)]
        blocks = lambda k: -(-k // bs)  # noqa: E731
        need = sum(blocks(p) for _, p in groups) + self.n + sum(blocks(p + o) - p // bs for (m, p), i0 in zip(groups, np.cumsum([0] + [m for m, _ in groups]))
                                                                for o in own[i0:i0 + m])
        ids = list(rng.permutation(need + 2))
        self.tables, self.meta, self.groups, self.keys = [], [], [], []
        elems = (need + 2, kv_heads, bs, D)
        k = rng.standard_normal(elems, dtype=np.float32) * spread
        v = rng.standard_normal(elems, dtype=np.float32)
        t = 0
        for m, p in groups:
            off = len(self.tables)
            prefix = [int(ids.pop()) for _ in range(blocks(p))]
            self.tables += prefix
            if m or p:
                self.groups.append([t, m, p, off])
            for _ in range(m):
                # Whole prefix blocks are shared; a last one that the prefix ends in is the member's own.
                mine = prefix[:p // bs] + [int(ids.pop()) for _ in range(blocks(p + own[t]) - p // bs)]
                at = len(self.tables)
                self.tables += mine
                c = p + own[t] if ctx is None else ctx[t]
                self.meta.append([t, 0 if t in idle else c, at, p])
                rows = [(prefix[j // bs], j % bs) if j < p else (mine[j // bs], j % bs) for j in range(c)]
                self.keys.append(rows)
                t += 1
        self.rows = rng.permutation(self.n)
        for i in range(self.n):
            self.meta[i][0] = int(self.rows[i])
        self.q, self.k, self.v = (f16_bits(x) for x in (rng.standard_normal((self.n, heads * D), dtype=np.float32) * spread, k, v))

    def max_own(self):
        return max([max(0, c - p) for _, c, _, p in self.meta] + [0])

    def oracle(self):
        """(values, tolerance) in 64 bits; idle rows NaN."""
        q, k, v = (bits_to_f32(x).astype(np.float64) for x in (self.q, self.k, self.v))
        H, KVH, D = self.heads, self.kv_heads, self.D
        out = np.full((self.n, H * D), np.nan)
        tol = np.zeros_like(out)
        for (row, c, _, _), where in zip(self.meta, self.keys):
            if c <= 0:
                continue
            b, s = (np.array(x) for x in zip(*where))
            K, V = k[b, :, s], v[b, :, s]  # [keys, kv heads, D]
            for h in range(H):
                g = h // (H // KVH)
                x = q[row, h * D:(h + 1) * D]
                logit = K[:, g] @ x / math.sqrt(D)
                size = (np.abs(K[:, g]) @ np.abs(x)).max() / math.sqrt(D)
                w = np.exp(logit - logit.max())
                w /= w.sum()
                o, a = w @ V[:, g], w @ np.abs(V[:, g])
                out[row, h * D:(h + 1) * D] = o
                tol[row, h * D:(h + 1) * D] = (2.0 ** -11 * np.abs(o) + 2.0 ** -25 + c * 2.0 ** -25 * np.abs(V[:, g]).max()
                                               + (2.0 ** -11 + 2 * (D + 2) * 2.0 ** -24 * size + 64 * 2.0 ** -24) * a)
        return out, tol


class Call:
    def __init__(self, torch, dev, case, hints=None, pad_q=0, pad_out=0, workspace=None):
        self.lib = _lib.lib()
        t = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a).view(dt)).to(dev)  # noqa: E731
        H, KVH, D, n = case.heads, case.kv_heads, case.D, case.n
        q = np.zeros((n, H * D + pad_q), np.uint16)
        q[:, :H * D] = case.q
        self.q, self.k, self.v = t(q, np.int16), t(case.k, np.int16), t(case.v, np.int16)
        self.meta = t(np.array(case.meta, np.int32).reshape(-1, 4), np.int32)
        self.groups = t(np.array(case.groups or [[0, 0, 0, 0]], np.int32), np.int32)
        self.tables = t(np.array(case.tables or [0], np.int32), np.int32)
        self.out = torch.full((n, H * D + pad_out), float("nan"), dtype=torch.float16, device=dev)
        ng = len(case.groups)
        hints = hints or (max([m for m, _ in [(g[1], g[2]) for g in case.groups]] + [0]), max([g[2] for g in case.groups] + [0]), case.max_own())
        size = self.lib.rh_shared_prefix_workspace(n, ng, *hints, H, KVH, D)
        self.workspace = torch.zeros(max(16, size), dtype=torch.uint8, device=dev) if workspace is None else workspace
        self.args = (self.q.data_ptr(), H * D + pad_q, self.k.data_ptr(), self.v.data_ptr(), self.meta.data_ptr(), self.groups.data_ptr(),
                     self.tables.data_ptr(), n, ng, *hints, H, KVH, D, case.bs, 1.0 / math.sqrt(D), self.workspace.data_ptr(), self.workspace.numel(),
                     self.out.data_ptr(), H * D + pad_out)

    def __call__(self, stream=None):
        _lib.check(self.lib.rh_shared_prefix_attention(*self.args, stream), "rh_shared_prefix_attention")
        return self.out


def check(torch, dev, case, **kw):
    print(f"shared prefix: groups={[(g[1], g[2]) for g in case.groups][:6]} n={case.n} {case.heads}/{case.kv_heads} D={case.D} bs={case.bs} {kw}", flush=True)
    call = Call(torch, dev, case, **kw)
    call()
    torch.cuda.synchronize()
    got = call.out.cpu().numpy().astype(np.float64)
    want, tol = case.oracle()
    width = case.heads * case.D
    assert np.isnan(got[:, width:]).all(), "written past the rows"
    got = got[:, :width]
    idle = np.isnan(want)
    assert np.isnan(got[idle]).all(), "an idle row was written"
    off = np.abs(got - want)[~idle]
    assert np.isfinite(off).all()
    assert (off <= tol[~idle]).all(), f"off by {off.max()}, {np.max(off / tol[~idle])} of the tolerance"
    return call


gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("D", [16, 32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (9, 3), (32, 4), (16, 1), (40, 1)])
def test_head_layouts(torch_mod, dev, heads, kv_heads, D):
    check(torch_mod, dev, Case([(5, 144), (2, 48)], [37, 1, 20], heads, kv_heads, D, seed=heads + D))


@gpu
@pytest.mark.parametrize("shared", [0, 1, 15, 16, 31, 32, 33, 255, 256, 257, 511, 1000, 2049])
def test_prefix_lengths(torch_mod, dev, shared):
    check(torch_mod, dev, Case([(7, shared)], [1, 16, 50], 8, 2, 64, seed=shared))


@gpu
@pytest.mark.parametrize("own", [1, 2, 31, 32, 33, 255, 257, 700, 1500])
@pytest.mark.parametrize("D", [64, 128])
def test_own_lengths(torch_mod, dev, own, D):
    check(torch_mod, dev, Case([(3, 80), (1, 0)], [own, max(1, own // 3)], 8, 2, D, seed=own))


@gpu
@pytest.mark.parametrize("members", [1, 2, 3, 8, 16, 33, 100])
@pytest.mark.parametrize("heads,kv_heads,D", [(9, 3, 64), (32, 8, 128)])
def test_group_sizes(torch_mod, dev, members, heads, kv_heads, D):
    check(torch_mod, dev, Case([(members, 300)], [5, 18], heads, kv_heads, D, seed=members))


@gpu
@pytest.mark.parametrize("bs", [1, 2, 8, 12, 16, 32, 64])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_block_sizes(torch_mod, dev, bs, D):
    """Prefixes that end inside a block, whose rest each member holds itself."""
    check(torch_mod, dev, Case([(4, 101), (3, 64)], [30, 3], 8, 2, D, bs=bs, seed=bs))


@gpu
def test_long_prefix_and_many_groups(torch_mod, dev):
    check(torch_mod, dev, Case([(20, 6001)], [9, 400], 8, 2, 128, seed=1))
    check(torch_mod, dev, Case([(3, 160 + 16 * i) for i in range(17)], [9, 40], 9, 3, 64, seed=2))


@gpu
def test_contexts_that_end_in_the_prefix_and_idle_tokens(torch_mod, dev):
    """A context of the prefix alone, one that ends inside it, of one key, and idle tokens."""
    ctx = [300, 299, 1, 17, 301, 350, 300, 256]
    check(torch_mod, dev, Case([(8, 300)], [60], 8, 2, 64, seed=3, ctx=ctx, idle=(6,)))
    check(torch_mod, dev, Case([(8, 300), (2, 0)], [60], 16, 2, 128, seed=4, idle=(0, 7, 9)))


@gpu
def test_large_scores_keep_their_order(torch_mod, dev):
    """Scores of some hundreds: weights fall to one key, in some slices far below fp16's range."""
    check(torch_mod, dev, Case([(6, 700)], [90], 8, 2, 64, seed=5, spread=8.0))


@gpu
@pytest.mark.parametrize("hints", [(1, 0, 0), (1, 64, 16), (100, 5000, 5000), (0, 0, 0), (1000000, 64, 16), (9, 3000000, 5000000)])
def test_hints_choose_speed_not_results(torch_mod, dev, hints):
    check(torch_mod, dev, Case([(9, 640), (5, 1200)], [40, 300], 9, 3, 64, seed=6), hints=hints)
    check(torch_mod, dev, Case([(9, 640), (5, 1200)], [40, 300], 16, 4, 128, seed=6), hints=hints)


@gpu
def test_the_most_tokens_of_a_call(torch_mod, dev):
    """65,536 (token, kv head) pairs, whose counters then lie next to each other."""
    check(torch_mod, dev, Case([(16, 16)] * 512, [1, 2, 3], 8, 8, 16, seed=11))


@gpu
def test_row_strides(torch_mod, dev):
    check(torch_mod, dev, Case([(5, 96)], [20], 8, 2, 64, seed=7), pad_q=8, pad_out=3)


@gpu
@pytest.mark.parametrize("members,shared,D", [(3, 50, 64), (9, 50, 64), (9, 50, 128), (3, 1100, 32), (40, 333, 64)])
def test_unwritten_slots_are_not_read(torch_mod, dev, members, shared, D):
    """NaN and infinities in the slots behind every context and every prefix."""
    case = Case([(members, shared)], [21, 2], 8, 2, D, seed=8)
    used = {w for rows in case.keys for w in rows}
    for b in range(case.k.shape[0]):
        for s in range(case.bs):
            if (b, s) not in used:
                case.k[b, :, s] = 0x7E00  # NaN
                case.v[b, :, s] = 0x7C00 if s % 2 else 0x7E00
    check(torch_mod, dev, case)


@gpu
@pytest.mark.parametrize("groups", [[(3, 80), (1, 0)], [(12, 300)]])
def test_cache_past_four_giga_values(torch_mod, dev, groups):
    """Blocks behind 2^32 values of K and of V: offsets need 64 bits."""
    torch = torch_mod
    case = Case(groups, [40, 5], 16, 8, 128, seed=14)
    call = Call(torch, dev, case)
    far, per = 262144 + 3, 8 * 16 * 128
    pools = [torch.empty((far + case.k.shape[0]) * per, dtype=torch.int16, device=dev) for _ in range(2)]
    for pool, small in zip(pools, (call.k, call.v)):
        pool[far * per:] = small.reshape(-1)
    args = list(call.args)
    args[2], args[3] = pools[0].data_ptr(), pools[1].data_ptr()
    call.tables += far
    _lib.check(call.lib.rh_shared_prefix_attention(*args, None))
    torch.cuda.synchronize()
    want, tol = case.oracle()
    assert (np.abs(call.out.double().cpu().numpy() - want) <= tol).all()


@gpu
def test_repeats_bit_for_bit_and_in_any_order(torch_mod, dev):
    """Two shapes in turn in one workspace: every call gives the bits of a first call."""
    torch = torch_mod
    a, b = Case([(12, 900)], [200, 3], 32, 4, 64, seed=9), Case([(3, 64), (5, 256)], [70], 8, 2, 128, seed=10)
    shared = torch.zeros(64 << 20, dtype=torch.uint8, device=dev)
    alone = [Call(torch, dev, c)().clone() for c in (a, b)]
    calls = [Call(torch, dev, c, workspace=shared) for c in (a, b)]
    for i in (0, 1, 1, 0, 0, 1):
        calls[i].out.fill_(float("nan"))
        assert torch.equal(calls[i](), alone[i])


@gpu
def test_batch_does_not_change_a_row(torch_mod, dev):
    """Agreement with rh_paged_decode_attention on the same contexts, within both tolerances."""
    torch = torch_mod
    case = Case([(6, 512)], [100, 33], 32, 4, 64, seed=11)
    got = check(torch, dev, case).out
    c = Call(torch, dev, case)
    H, KVH, D, n = case.heads, case.kv_heads, case.D, case.n
    parts = -(-max(m[1] for m in case.meta) // 512)
    part_o, part_ml = torch.empty(n * H * parts * D, device=dev), torch.empty(n * H * parts * 2, device=dev)
    counters = torch.zeros(n * KVH, dtype=torch.int32, device=dev)
    # The members' own tables hold the whole prefix too (it ends on a block).
    _lib.check(c.lib.rh_paged_decode_attention(c.q.data_ptr(), H * D, c.k.data_ptr(), c.v.data_ptr(), c.meta.data_ptr(), c.tables.data_ptr(), n, H, KVH, D,
                                               16, 512, parts, 1.0 / math.sqrt(D), part_o.data_ptr(), part_ml.data_ptr(), counters.data_ptr(),
                                               c.out.data_ptr(), H * D, None))
    torch.cuda.synchronize()
    _, tol = case.oracle()
    assert (np.abs((got.double() - c.out.double()).cpu().numpy()) <= 2 * tol).all()


@gpu
def test_graph_replays_and_streams(torch_mod, dev):
    """Captured on a stream of its own, replayed with new queries and lengths, eager work between."""
    torch = torch_mod
    case = Case([(9, 400)], [130], 32, 8, 128, seed=12)
    call = Call(torch, dev, case, hints=(9, 400, 130))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call(s.cuda_stream)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call(torch.cuda.current_stream().cuda_stream)
    for step in range(4):
        call.q.copy_(torch.roll(call.q, 1, 0))
        call.meta[:, 1] -= step
        call.out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        got = call.out.clone()
        call.out.fill_(float("nan"))
        assert torch.equal(call().clone(), got)
        torch.cuda.synchronize()


# ---- groups of a step, found on the host ---------------------------------------------------------------

def groups_of(tokens, tables, bs, least):
    t, tab = np.ascontiguousarray(tokens, np.int32), np.ascontiguousarray(tables, np.int32)
    n = len(t)
    meta, groups, limits = np.full((n, 4), -9, np.int32), np.full((n, 4), -9, np.int32), np.full(3, -9, np.int32)
    got = _lib.lib().rh_shared_prefix_groups(t.ctypes.data, tab.ctypes.data, n, bs, least, meta.ctypes.data, groups.ctypes.data, limits.ctypes.data)
    assert got >= 0, _lib.last_error()
    assert (groups[got:] == -9).all()
    return meta, groups[:got], limits


def saved_at_most(rows, ctx, bs, least):
    """The most blocks that any partition into groups saves, by trying all of them."""
    def partitions(items):
        if not items:
            yield []
            return
        for rest in partitions(items[1:]):
            yield [[items[0]]] + rest
            for k in range(len(rest)):
                yield rest[:k] + [[items[0]] + rest[k]] + rest[k + 1:]

    def common(group):
        n = min(ctx[i] // bs for i in group)
        k = 0
        while k < n and len({rows[i][k] for i in group}) == 1:
            k += 1
        return k if k * bs >= max(least, 1) else 0
    return max(sum((len(g) - 1) * common(g) for g in p) for p in partitions(list(range(len(rows)))))


@pytest.mark.parametrize("seed", range(12))
def test_groups_save_the_most_and_share_what_they_say(seed):
    r = np.random.default_rng(seed)
    bs, n, least = int(r.choice([1, 4, 16])), int(r.integers(1, 8)), int(r.choice([0, 5, 33]))
    prompts = [list(r.integers(0, 3, 6)) for _ in range(2)]
    rows, ctx, tables, tokens = [], [], [], []
    for i in range(n):
        own = [int(x) for x in r.integers(0, 3, 7)]
        cut = int(r.integers(0, 7))
        rows.append([int(x) for x in prompts[int(r.integers(0, 2))][:cut]] + own[cut:])
        ctx.append(int(r.integers(0, 7 * bs + 1)))
        tokens.append([10 + i, ctx[i], len(tables), 77])
        tables += rows[i]
    meta, groups, limits = groups_of(tokens, tables, bs, least)
    assert sorted(meta[:, 0]) == [10 + i for i in range(n)]
    grouped = np.zeros(n, bool)
    for first, members, shared, off in groups:
        assert members > 1 and shared % bs == 0 and shared >= max(1, least)
        grouped[first:first + members] = True
        for t in meta[first:first + members]:
            i = t[0] - 10
            assert t[3] == shared and t[1] == ctx[i] >= shared and t[2] == tokens[i][2]
            assert tables[off:off + shared // bs] == rows[i][:shared // bs]
    assert (meta[~grouped, 3] == 0).all()
    assert sum((m - 1) * s for _, m, s, _ in groups) == saved_at_most(rows, ctx, bs, least) * bs
    assert limits.tolist() == [max([g[1] for g in groups], default=0), max([g[2] for g in groups], default=0), max(0, *(meta[:, 1] - meta[:, 3]))]


def test_groups_of_nothing_and_refusals():
    lib = _lib.lib()
    lim = np.zeros(3, np.int32)
    assert lib.rh_shared_prefix_groups(None, None, 0, 16, 0, None, None, lim.ctypes.data) == 0
    for args in ((None, None, -1, 16, 0, None, None, lim.ctypes.data), (None, None, 0, 0, 0, None, None, lim.ctypes.data),
                 (None, None, 0, 16, -1, None, None, lim.ctypes.data), (None, None, 3, 16, 0, None, None, lim.ctypes.data), (None, None, 0, 16, 0, None, None, None)):
        assert lib.rh_shared_prefix_groups(*args) < 0 and "shared prefix groups" in _lib.last_error()


@gpu
def test_groups_from_the_host_give_the_decode_kernels_attention(torch_mod, dev):
    """Ungrouped descriptors through rh_shared_prefix_groups: the same attention as without sharing."""
    case = Case([(5, 320), (1, 0), (4, 96), (2, 16)], [33, 150, 7], 32, 4, 64, seed=13)
    tokens = [[m[0], m[1], m[2], 0] for m in np.random.default_rng(1).permutation(case.meta).tolist()]
    meta, groups, limits = groups_of(tokens, case.tables, case.bs, 32)
    assert sorted((g[1], g[2]) for g in groups) == [(4, 96), (5, 320)]
    case.meta, case.groups = meta.tolist(), groups.tolist()
    want, tol = Case([(5, 320), (1, 0), (4, 96), (2, 16)], [33, 150, 7], 32, 4, 64, seed=13).oracle()
    call = Call(torch_mod, dev, case, hints=tuple(int(x) for x in limits))
    call()
    torch_mod.cuda.synchronize()
    assert (np.abs(call.out.double().cpu().numpy() - want) <= tol).all()


# ---- refusals (nothing is launched: the CPU suffices) ------------------------------------------------

GOOD = dict(q=16, q_row_stride=256, kpool=16, vpool=16, dec_meta=16, groups=16, tables=16, n_dec=4, n_groups=1, max_members=4, max_shared=64, max_own=16,
            heads=4, kv_heads=2, head_dim=64, block_size=16, scale=0.125, workspace=16, workspace_bytes=1 << 40, out=16, out_row_stride=256, stream=None)


@pytest.mark.parametrize("change,message", [
    ({"n_dec": -1}, "bad sizes"), ({"n_groups": -1}, "bad sizes"), ({"max_members": -1}, "bad sizes"), ({"max_own": -1}, "bad sizes"),
    ({"max_shared": -5}, "bad sizes"), ({"heads": 5}, "head counts"), ({"kv_heads": 0}, "head counts"), ({"head_dim": 48}, "head_dim"),
    ({"block_size": 0}, "block size"), ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"q": None}, "missing pointer"), ({"groups": None}, "missing pointer"), ({"tables": None}, "missing pointer"),
    ({"out": None}, "missing pointer"), ({"q_row_stride": 260}, "16-byte"), ({"out_row_stride": 255}, "out rows"), ({"q": 8}, "aligned"),
    ({"dec_meta": 20}, "aligned"), ({"workspace": None}, "workspace"), ({"workspace": 24}, "workspace"), ({"workspace_bytes": 64}, "workspace"),
    ({"max_shared": (1 << 30) + 1}, "2^30"), ({"max_own": (1 << 31) - 1}, "2^30"), ({"n_dec": 40000}, "65536"), ({"scale": 3e38}, "scale")])
def test_refusals(change, message):
    lib = _lib.lib()
    assert lib.rh_shared_prefix_attention(*{**GOOD, **change}.values()) != 0
    assert message in _lib.last_error()


@pytest.mark.parametrize("n,shared,own,heads,kv_heads,D,pays", [
    (4, 4096, 300, 32, 8, 128, 0), (32, 1024, 300, 32, 8, 128, 1), (64, 16384, 1000, 32, 8, 128, 1), (32, 2048, 300, 32, 4, 64, 0), (64, 2048, 500, 32, 4, 64, 1),
    (2, 512, 40, 9, 3, 64, 0), (2, 4096, 100, 16, 1, 128, 1), (64, 0, 9000, 32, 8, 128, 0), (0, 512, 40, 9, 3, 64, 0), (4, 512, 40, 9, 2, 64, 0)])
def test_sharing_pays_where_it_is_measured_faster(n, shared, own, heads, kv_heads, D, pays):
    assert _lib.lib().rh_shared_prefix_pays(n, shared, own, heads, kv_heads, D) == pays


def test_nothing_to_do_is_not_an_error():
    assert _lib.lib().rh_shared_prefix_attention(*{**GOOD, "n_dec": 0, "q": None}.values()) == 0
    assert _lib.lib().rh_shared_prefix_workspace(0, 0, 0, 0, 0, 8, 2, 64) == 0
    assert _lib.lib().rh_shared_prefix_workspace(4, 1, 4, 64, 16, 9, 2, 64) == 0
