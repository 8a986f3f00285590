"""Step tables, q/k norm with rotation and cache write, and logits processing, each against its
formula in 64 bits (whole numbers: equal), and their refusals (on the CPU)."""
import numpy as np
import pytest

from relay_amd import _lib

gpu = pytest.mark.gpu


def dev_of(torch, dev, a, dt=None):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a if dt is None else a.astype(dt)).to(dev)


def ptr(t):
    return 0 if t is None else t.data_ptr()


# ---- block tables and slot maps ----------------------------------------------------------------------

ROWS_FULL, NO_BLOCKS, TABLE_FULL, BAD_LENGTH = 1, 2, 4, 8


def tables_oracle(cached, fresh, shared, group_seqs, B, tables, free, max_rows):
    n, stride = tables.shape
    held, want = -(-cached // B), -(-(cached + fresh) // B)
    status = (ROWS_FULL if fresh.sum() > max_rows else 0) | (NO_BLOCKS if (want - held).sum() > len(free) else 0) | \
        (TABLE_FULL if (want > stride).any() else 0)
    tables, free = tables.copy(), list(free)
    off = np.zeros(n + 1, int)
    rows = []
    if not status:
        off[1:] = np.cumsum(fresh)
        for s in range(n):
            for j in range(held[s], want[s]):
                tables[s, j] = free.pop()
            rows += [(s, p) for p in range(cached[s], cached[s] + fresh[s])]
    pos, seq, slot = np.zeros(max_rows, int), np.zeros(max_rows, int), np.full(max_rows, -1)
    meta = np.array([[t, 0, 0, 0] for t in range(max_rows)]).reshape(-1, 4)
    for t, (s, p) in enumerate(rows):
        pos[t], seq[t], slot[t] = p, s, tables[s, p // B] * B + p % B
        meta[t] = [t, p + 1, s * stride, shared[s]]
    groups = [[off[f], off[f + m] - off[f], shared[f] if m else 0, f * stride if m else 0] for f, m in group_seqs] if not status else \
        [[0, 0, 0, 0] for _ in group_seqs]
    return {"tables": tables, "row_off": off, "last_row": np.where((np.diff(off) > 0), off[1:] - 1, 0), "table_off": np.arange(n) * stride, "pos": pos,
            "seq": seq, "slot": slot, "meta": meta, "groups": np.array(groups).reshape(-1, 4),
            "totals": np.array([len(rows), int((want - held).sum()) if not status else 0, len(free), status])}


def tables_case(seed, n, ctx, chunk, B, ng, extra=7, short=0, narrow=0, waits=0.2):
    r = np.random.default_rng(seed)
    cached = r.integers(0, ctx + 1, size=n)
    fresh = np.where(r.random(n) < 0.5, 1, r.integers(0, chunk + 1, size=n))
    fresh[r.random(n) < waits] = 0
    held, want = -(-cached // B), -(-(cached + fresh) // B)
    stride = int(max(want.max(initial=0), held.max(initial=0), 1)) + 2 - narrow
    ids = r.permutation(int(want.sum()) + 5)
    tables = np.full((n, stride), -7)
    at = 0
    for s in range(n):
        k = min(held[s], stride)
        tables[s, :k] = ids[at:at + k]
        at += k
    free = ids[at:at + int((want - held).sum()) + 2 - short]
    cuts = np.sort(r.integers(0, n + 1, size=2 * ng)).reshape(-1, 2)
    groups = [(int(a), int(b - a)) for a, b in cuts]
    shared = np.zeros(n, int)
    for f, m in groups:
        shared[f:f + m] = int(r.integers(0, ctx + 1))
    return cached, fresh, shared, groups, B, tables, free, int(fresh.sum()) + extra


def run_tables(torch, dev, cached, fresh, shared, groups, B, tables, free, max_rows, with_shared=True, carry=False, count=None):
    n, stride = tables.shape
    i = lambda a: dev_of(torch, dev, a, np.int32)  # noqa: E731
    e = lambda *s: torch.full(s, -99, dtype=torch.int32, device=dev)  # noqa: E731
    out = {"tables": i(tables), "row_off": e(n + 1), "last_row": e(max(n, 1)), "table_off": e(max(n, 1)), "pos": e(max_rows + 1), "seq": e(max_rows + 1),
           "slot": e(max_rows + 1), "meta": e(max_rows + 1, 4), "groups": e(len(groups) + 1, 4), "totals": e(4)}
    c, f, s, g, fb, fc = i(cached), i(fresh), i(shared), i(np.array(groups).reshape(-1, 2)), i(np.append(free, -1)), i([len(free) if count is None else count])
    if carry:
        out["totals"][2] = len(free)
    print(f"step tables: n={n} rows={max_rows} B={B} groups={len(groups)} stride={stride}", flush=True)
    _lib.check(_lib.lib().rh_step_tables(ptr(c), ptr(f), ptr(s) if with_shared else None, n, ptr(g), len(groups), B, ptr(out["tables"]), stride, ptr(fb),
                                         out["totals"].data_ptr() + 8 if carry else ptr(fc), max_rows, ptr(out["row_off"]), ptr(out["last_row"]),
                                         ptr(out["table_off"]), ptr(out["pos"]), ptr(out["seq"]), ptr(out["slot"]), ptr(out["meta"]), ptr(out["groups"]),
                                         ptr(out["totals"]), None))
    torch.cuda.synchronize()
    got = {k: v.cpu().numpy() for k, v in out.items()}
    for k, size in (("pos", max_rows), ("seq", max_rows), ("slot", max_rows), ("meta", max_rows), ("groups", len(groups)), ("last_row", n), ("table_off", n)):
        assert (got[k][size:] == -99).all(), f"{k}: written past its end"
        got[k] = got[k][:size]
    assert np.array_equal(c.cpu().numpy(), cached) and np.array_equal(f.cpu().numpy(), fresh)
    return got


def same(got, want):
    for k, w in want.items():
        assert np.array_equal(got[k], w), f"{k}: {got[k]} for {w}"


@gpu
@pytest.mark.parametrize("seed,n,ctx,chunk,B,ng", [
    (0, 1, 0, 1, 16, 0), (1, 1, 100, 1, 16, 1), (2, 48, 300, 1, 16, 2), (3, 7, 64, 40, 12, 3), (4, 511, 200, 90, 16, 5), (5, 1023, 50, 3, 1, 2),
    (6, 1024, 50, 3, 32, 2), (7, 1025, 50, 3, 8, 2), (8, 3000, 40, 5, 16, 1100), (9, 3, 5000, 9000, 16, 1), (10, 2500, 9, 20, 64, 0)])
def test_step_tables(torch_mod, dev, seed, n, ctx, chunk, B, ng):
    case = tables_case(seed, n, ctx, chunk, B, ng)
    same(run_tables(torch_mod, dev, *case), tables_oracle(*case))


@gpu
def test_step_tables_with_no_rows_or_no_sequences(torch_mod, dev):
    for n, extra in ((5, 0), (5, 4), (1, 1)):
        c = list(tables_case(20, n, 60, 1, 16, 1, extra=extra))
        c[1] = np.zeros(n, int)  # every sequence waits
        c[-1] = extra
        same(run_tables(torch_mod, dev, *c), tables_oracle(*c))
    got = run_tables(torch_mod, dev, np.zeros(0, int), np.zeros(0, int), np.zeros(0, int), [], 16, np.zeros((0, 4), int), np.arange(3), 5)
    assert (got["slot"] == -1).all() and (got["meta"][:, 1] == 0).all() and got["totals"].tolist() == [0, 0, 3, 0] and got["row_off"].tolist() == [0]


@gpu
def test_step_tables_without_shared_and_with_carried_stack(torch_mod, dev):
    case = tables_case(21, 30, 100, 9, 16, 2)
    want = tables_oracle(case[0], case[1], np.zeros(30, int), *case[3:])
    same(run_tables(torch_mod, dev, *case, with_shared=False), want)
    same(run_tables(torch_mod, dev, *case, carry=True), tables_oracle(*case))


@gpu
@pytest.mark.parametrize("max_rows", [512, 513, 5000])
def test_step_tables_of_idle_rows(torch_mod, dev, max_rows):
    got = run_tables(torch_mod, dev, np.zeros(0, int), np.zeros(0, int), np.zeros(0, int), [], 16, np.zeros((0, 4), int), np.arange(3), max_rows)
    assert (got["slot"] == -1).all() and (got["meta"][:, 1] == 0).all() and got["totals"].tolist() == [0, 0, 3, 0] and got["row_off"].tolist() == [0]
    c = list(tables_case(24, 6, 60, 1, 16, 2))
    c[-1] = max_rows
    same(run_tables(torch_mod, dev, *c), tables_oracle(*c))
    c[1] = np.zeros(6, int)
    same(run_tables(torch_mod, dev, *c), tables_oracle(*c))


@gpu
@pytest.mark.parametrize("seed,n,ctx,chunk,B,ng,carry", [
    (30, 511, 200, 90, 16, 5, True), (31, 3, 5000, 9000, 16, 1, True), (32, 1500, 40, 5, 16, 3, True), (33, 200, 60, 30, 16, 2, True),
    (34, 4096, 20, 3, 16, 4, False), (35, 4097, 20, 3, 16, 4, False), (36, 4097, 20, 30, 12, 2, True), (37, 257, 60, 4, 16, 1, False)])
def test_step_tables_of_large_steps(torch_mod, dev, seed, n, ctx, chunk, B, ng, carry):
    """More sequences than a workgroup keeps, and a stack count that lies in the totals."""
    case = tables_case(seed, n, ctx, chunk, B, ng)
    same(run_tables(torch_mod, dev, *case, carry=carry), tables_oracle(*case))
    case = tables_case(seed, n, ctx, chunk, B, ng, short=3, waits=0.0)
    same(run_tables(torch_mod, dev, *case, carry=carry), tables_oracle(*case))


@gpu
@pytest.mark.parametrize("change,status", [({"extra": -1}, ROWS_FULL), ({"short": 3}, NO_BLOCKS), ({"narrow": 3}, TABLE_FULL),
                                           ({"extra": -1, "short": 3}, ROWS_FULL | NO_BLOCKS)])
@pytest.mark.parametrize("n", [40, 1500])
def test_step_tables_that_do_not_fit_change_nothing(torch_mod, dev, n, change, status):
    case = tables_case(22, n, 100, 9, 16, 2, waits=0.0, **change)
    want = tables_oracle(*case)
    assert want["totals"][3] == status
    same(run_tables(torch_mod, dev, *case), want)


@gpu
@pytest.mark.parametrize("which,value", [("cached", -1), ("fresh", -3), ("cached", (1 << 30) - 1), ("fresh", 2 ** 31 - 1), ("shared", -1),
                                         ("groups", (-1, 2)), ("groups", (3, 99)), ("groups", (2 ** 31 - 1, 2 ** 31 - 1)), ("free", -2)])
def test_step_tables_with_bad_lengths_change_nothing(torch_mod, dev, which, value):
    case = list(tables_case(23, 20, 100, 9, 16, 1))
    good = tables_oracle(*case)
    if which == "groups":
        case[3] = [value]
    elif which != "free":
        case[1][7] = 1
        case[{"cached": 0, "fresh": 1, "shared": 2}[which]][7] = value
    got = run_tables(torch_mod, dev, *case, count=value if which == "free" else None)
    assert got["totals"][0] == 0 and got["totals"][1] == 0 and got["totals"][3] & BAD_LENGTH
    assert np.array_equal(got["tables"], case[5]) and (got["slot"] == -1).all() and (got["meta"][:, 1:] == 0).all() and (got["row_off"] == 0).all()
    assert (got["groups"] == 0).all() and (got["last_row"] == 0).all()
    assert np.array_equal(got["table_off"], good["table_off"])


# ---- norm of q and k, rotation, cache write ------------------------------------------------------------

class QkCase:
    def __init__(self, T, heads, kv_heads, D, bs=16, planes=1, bias=False, scale=False, seed=0, idle=(), top=4096, q_scale=0.25, spread=1.0):
        r = np.random.default_rng(seed)
        self.T, self.heads, self.kv_heads, self.D, self.bs, self.planes, self.q_scale = T, heads, kv_heads, D, bs, planes, q_scale
        W = (heads + 2 * kv_heads) * D
        f = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
        self.qkv = f(planes, T, W) * np.float32(spread)
        self.bias = f(W) if bias else None
        self.scale = r.uniform(0.5, 2, W).astype(np.float32) if scale else None
        self.wq, self.wk = 1 + np.float32(0.3) * f(D), 1 + np.float32(0.3) * f(D)
        self.inv_freq = (10000.0 ** (-np.arange(0, D, 2) / D)).astype(np.float32)
        self.pos = r.integers(0, top, size=T)
        self.nb = -(-T // bs) + 3
        self.slot = r.permutation(self.nb * bs)[:T]
        self.slot[list(idle)] = -1
        self.pool = r.standard_normal((2, self.nb, kv_heads, bs, D)).astype(np.float16)
        self.q0 = r.standard_normal((T, heads * D)).astype(np.float16)
        self.eps = 1e-6

    def oracle(self):
        """{name: (values, tolerance)}: fp16's rounding, and fp32 sums: planes + scale + bias, the mean's D products and a few roundings."""
        H, KVH, D, T = self.heads, self.kv_heads, self.D, self.T
        x, size = self.qkv.astype(np.float64).sum(0), np.abs(self.qkv).astype(np.float64).sum(0)
        if self.scale is not None:
            x, size = x * self.scale, size * self.scale
        if self.bias is not None:
            x, size = x + self.bias, size + np.abs(self.bias)
        x, size = x.reshape(T, -1, D), size.reshape(T, -1, D)
        first = (self.planes + 2) * 2.0 ** -24 * size  # of x
        qk, e = x[:, :H + KVH], first[:, :H + KVH]
        w = np.concatenate([np.tile(self.wq, (H, 1)), np.tile(self.wk, (KVH, 1))]).astype(np.float64)
        rms = np.sqrt((qk ** 2).mean(-1, keepdims=True) + self.eps)
        # The mean is off by its sum's D + 3 roundings and by x's own error, which moves all of a head.
        rel = (D + 8) * 2.0 ** -24 + (np.abs(qk) * e).mean(-1, keepdims=True) / rms ** 2
        y, ye = qk / rms * w, (e / rms + np.abs(qk) / rms * rel) * np.abs(w)
        angle = self.pos[:, None] * self.inv_freq.astype(np.float64)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        lo, hi, le, he = y[..., :D // 2], y[..., D // 2:], ye[..., :D // 2], ye[..., D // 2:]
        z = np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)
        # cos and sin of a turn rounded to fp32 (2^-25 of a turn) and their own rounding: 2^-21 in all.
        ze = np.concatenate([le + he, le + he], -1) + 2.0 ** -21 * np.concatenate([np.abs(lo) + np.abs(hi)] * 2, -1)
        half = lambda v, err: (v, err + 2.0 ** -11 * (np.abs(v) + err) + 2.0 ** -25)  # noqa: E731
        out = {"q": half((z[:, :H] * self.q_scale).reshape(T, -1), (ze[:, :H] * self.q_scale).reshape(T, -1))}
        for i, (v, err) in enumerate(((z[:, H:], ze[:, H:]), (x[:, H + KVH:], first[:, H + KVH:]))):
            pool, tol = self.pool[i].astype(np.float64), np.zeros(self.pool[i].shape)
            live = self.slot >= 0
            b, at = self.slot[live] // self.bs, self.slot[live] % self.bs
            pool[b, :, at], tol[b, :, at] = half(v[live], err[live])
            out["kv"[i]] = (pool, tol)
        idle = self.slot < 0
        out["q"][0][idle], out["q"][1][idle] = self.q0[idle], 0
        return out


def check_qk(torch, dev, case, stream=None):
    d = lambda a: None if a is None else dev_of(torch, dev, a)  # noqa: E731
    i = lambda a: dev_of(torch, dev, a, np.int32)  # noqa: E731
    t = [d(case.qkv), d(case.scale), d(case.bias), d(case.wq), d(case.wk), d(case.inv_freq), i(case.pos), i(case.slot), d(case.pool[0]), d(case.pool[1]),
         d(case.q0)]
    print(f"qk norm: T={case.T} {case.heads}/{case.kv_heads} D={case.D} bs={case.bs} planes={case.planes}", flush=True)
    _lib.check(_lib.lib().rh_qk_norm_to_cache(ptr(t[0]), case.planes, ptr(t[1]), case.T, ptr(t[2]), ptr(t[3]), ptr(t[4]), case.eps, ptr(t[5]), ptr(t[6]),
                                              ptr(t[7]), ptr(t[8]), ptr(t[9]), ptr(t[10]), case.q_scale, case.heads, case.kv_heads, case.D, case.bs, stream))
    torch.cuda.synchronize()
    for name, got in zip("kvq", t[8:]):
        want, tol = case.oracle()[name]
        got = got.cpu().numpy().astype(np.float64)
        off = np.abs(got - want)
        assert (off <= tol).all(), f"{name} off by {off.max()}"


@gpu
@pytest.mark.parametrize("D", [8, 16, 24, 32, 40, 64, 80, 96, 128, 192, 256, 320, 512])
def test_qk_norm_head_sizes(torch_mod, dev, D):
    check_qk(torch_mod, dev, QkCase(5, 6, 2, D, seed=D))


@gpu
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (9, 3), (32, 4), (32, 8), (40, 5), (3, 3)])
@pytest.mark.parametrize("T", [1, 3, 130])
def test_qk_norm_head_layouts(torch_mod, dev, heads, kv_heads, T):
    check_qk(torch_mod, dev, QkCase(T, heads, kv_heads, 64, seed=heads + T, idle=(T - 1,) if T > 2 else ()))
    check_qk(torch_mod, dev, QkCase(T, heads, kv_heads, 128, seed=heads + T, bias=True))


@gpu
@pytest.mark.parametrize("planes", [1, 2, 3, 8])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scale", [False, True])
def test_qk_norm_planes_scale_bias(torch_mod, dev, planes, bias, scale):
    check_qk(torch_mod, dev, QkCase(33, 9, 3, 64, planes=planes, bias=bias, scale=scale, seed=planes, idle=(0, 7)))


@gpu
@pytest.mark.parametrize("bs", [1, 12, 16, 64])
def test_qk_norm_block_sizes(torch_mod, dev, bs):
    check_qk(torch_mod, dev, QkCase(50, 8, 2, 64, bs=bs, seed=bs))


@gpu
def test_qk_norm_far_positions_and_extremes(torch_mod, dev):
    check_qk(torch_mod, dev, QkCase(64, 8, 2, 128, top=1 << 24, seed=1))
    check_qk(torch_mod, dev, QkCase(9, 8, 2, 64, spread=1e-4, seed=2))   # eps counts
    check_qk(torch_mod, dev, QkCase(9, 8, 2, 64, spread=300.0, seed=3))
    case = QkCase(4, 8, 2, 64, seed=4)
    case.qkv[:] = 0  # a row of zeros has no direction: zeros
    check_qk(torch_mod, dev, case)


@gpu
def test_qk_norm_into_a_cache_past_four_giga_values(torch_mod, dev):
    """A slot behind 2^32 values of each pool."""
    torch = torch_mod
    case = QkCase(3, 9, 8, 128, seed=7)
    far = 262144 + 5
    pools = [torch.empty(far + case.nb, 8, 16, 128, dtype=torch.float16, device=dev) for _ in range(2)]
    for pool, small in zip(pools, case.pool):
        pool[far:] = dev_of(torch, dev, small)
    d = lambda a: dev_of(torch, dev, a)  # noqa: E731
    t = [d(case.qkv), d(case.wq), d(case.wk), d(case.inv_freq), dev_of(torch, dev, case.pos, np.int32), dev_of(torch, dev, case.slot + far * 16, np.int32), d(case.q0)]
    _lib.check(_lib.lib().rh_qk_norm_to_cache(ptr(t[0]), 1, None, 3, None, ptr(t[1]), ptr(t[2]), case.eps, ptr(t[3]), ptr(t[4]), ptr(t[5]), ptr(pools[0]),
                                              ptr(pools[1]), ptr(t[6]), case.q_scale, 9, 8, 128, 16, None))
    torch.cuda.synchronize()
    for name, pool in zip("kv", pools):
        want, tol = case.oracle()[name]
        assert (np.abs(pool[far:].cpu().numpy().astype(np.float64) - want) <= tol).all()


@gpu
def test_qk_norm_many_rows(torch_mod, dev):
    check_qk(torch_mod, dev, QkCase(1501, 8, 2, 64, seed=5, idle=(3, 1500)))
    check_qk(torch_mod, dev, QkCase(700, 32, 8, 128, seed=6, planes=2))


# ---- penalties, biases and masks --------------------------------------------------------------------------

class LogitCase:
    def __init__(self, rows, vocab, history=0, biases=0, masks=0, seed=0, ld=None, prompt=True, allowed=0.3):
        r = np.random.default_rng(seed)
        self.rows, self.vocab, self.ld = rows, vocab, ld or vocab
        self.logits = np.full((rows, self.ld), 77, np.float32)
        self.logits[:, :vocab] = r.standard_normal((rows, vocab)) * 4
        self.history = None if not history else (vocab * r.random((rows, history)) ** 4).astype(np.int64).clip(0, vocab - 1)
        self.history_len = r.integers(0, history + 1, size=rows)
        self.prompt_len = (self.history_len * r.random(rows)).astype(int) if prompt else None
        self.repetition, self.frequency, self.presence = (x.astype(np.float32) for x in (r.uniform(0.8, 1.5, rows), r.uniform(-0.5, 0.5, rows), r.uniform(-1, 1, rows)))
        self.bias_tokens = None if not biases else r.integers(0, vocab, size=(rows, biases))
        self.bias_values = r.standard_normal((rows, max(1, biases))).astype(np.float32) * 5
        self.bias_len = r.integers(0, biases + 1, size=rows)
        self.masks = None if not masks else r.random((masks, vocab)) < allowed
        self.mask_of = r.integers(-1, masks, size=rows) if masks else None

    def oracle(self):
        """The formula with each step in fp32 (the kernel's own steps), and in 64 bits with its tolerance: 5 roundings of the parts' sizes."""
        x32, x64 = self.logits[:, :self.vocab].copy(), self.logits[:, :self.vocab].astype(np.float64)
        tol = np.zeros_like(x64)
        for r in range(self.rows):
            if self.history is not None:
                n = min(max(self.history_len[r], 0), self.history.shape[1])
                p = 0 if self.prompt_len is None else self.prompt_len[r]
                said = self.history[r, :n]
                ok = (said >= 0) & (said < self.vocab)
                seen = np.unique(said[ok])
                rep = self.repetition[r] if self.repetition is not None else np.float32(1)
                f, q = (np.float32(0) if v is None else v[r] for v in (self.frequency, self.presence))
                x32[r, seen] = np.where(x32[r, seen] > 0, x32[r, seen] / rep, x32[r, seen] * rep)
                x64[r, seen] = np.where(x64[r, seen] > 0, x64[r, seen] / float(rep), x64[r, seen] * float(rep))
                out, count = np.unique(said[p:][ok[p:]], return_counts=True)
                x32[r, out] = x32[r, out] - f * count.astype(np.float32) - q
                x64[r, out] -= float(f) * count + float(q)
                tol[r, seen] += 2.0 ** -24 * 5 * np.abs(x64[r, seen])
                tol[r, out] += 2.0 ** -24 * 5 * (np.abs(self.logits[r, out] * max(rep, 1 / rep)) + np.abs(f) * count + np.abs(q))
            if self.bias_tokens is not None:
                named = {}
                for j in range(min(max(self.bias_len[r], 0), self.bias_tokens.shape[1])):
                    named[int(self.bias_tokens[r, j])] = self.bias_values[r, j]
                for t, v in named.items():
                    if 0 <= t < self.vocab:
                        tol[r, t] += 2.0 ** -24 * 5 * (np.abs(x64[r, t]) + abs(float(v)))
                        x32[r, t] += v
                        x64[r, t] += float(v)
            m = None if self.masks is None else (r if self.mask_of is None else self.mask_of[r])
            if m is not None and m >= 0:
                x32[r, ~self.masks[m]] = x64[r, ~self.masks[m]] = -np.inf
                tol[r, ~self.masks[m]] = 0
        return x32, x64, tol

    def call(self, torch, dev, in_place=False, out_ld=None, next_=True, workspace=None, shift=0, stream=None):
        i = lambda a: None if a is None else dev_of(torch, dev, a, np.int32)  # noqa: E731
        d = lambda a: None if a is None else dev_of(torch, dev, a)  # noqa: E731
        words = -(-self.vocab // 32) + 1
        masks = None
        if self.masks is not None:
            bits = np.zeros((len(self.masks), words * 32), bool)
            bits[:, :self.vocab] = self.masks
            bits[:, self.vocab:] = True
            masks = torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32)).to(dev)
        flat = torch.full((self.rows * self.ld + 8,), 77.0, device=dev)
        logits = flat[shift:shift + self.rows * self.ld].view(self.rows, self.ld)
        logits.copy_(d(self.logits))
        out_ld = self.ld if in_place else out_ld or self.vocab
        out = logits if in_place else torch.full((self.rows * out_ld + 8,), 55.0, device=dev)[shift:shift + self.rows * out_ld].view(self.rows, out_ld)
        nxt = torch.full((self.rows + 1,), -99, dtype=torch.int32, device=dev)
        L = _lib.lib()
        size = L.rh_process_logits_workspace(self.rows, self.vocab)
        ws = torch.zeros(size, dtype=torch.uint8, device=dev) if workspace is None else workspace
        t = [i(self.history), i(self.history_len), i(self.prompt_len), d(self.repetition), d(self.frequency), d(self.presence), i(self.bias_tokens),
             d(self.bias_values), i(self.bias_len), masks, i(self.mask_of)]
        h = self.history is not None
        print(f"logits: rows={self.rows} vocab={self.vocab} ld={self.ld}/{out_ld} shift={shift} history={0 if not h else self.history.shape[1]}", flush=True)
        self.keep = (flat, t, ws)
        args = (ptr(logits), self.ld, self.rows, self.vocab, ptr(t[0]), self.history.shape[1] if h else 0, ptr(t[1]), ptr(t[2]) if h else 0,
                ptr(t[3]) if h else 0, ptr(t[4]) if h else 0, ptr(t[5]) if h else 0, ptr(t[6]), ptr(t[7]), 0 if t[6] is None else t[6].shape[1], ptr(t[8]),
                ptr(masks), words, ptr(t[10]), ptr(out), out_ld, ptr(nxt) if next_ else 0, ptr(ws), ws.numel())
        return args, out, nxt, ws, logits


def check_logits(torch, dev, case, **kw):
    args, out, nxt, ws, logits = case.call(torch, dev, **kw)
    _lib.check(_lib.lib().rh_process_logits(*args, None))
    torch.cuda.synchronize()
    x32, x64, tol = case.oracle()
    full = out.cpu().numpy()
    got = full[:, :case.vocab]
    assert (full[:, case.vocab:] == (77 if kw.get("in_place") else 55)).all(), "written past the rows"
    if not kw.get("in_place"):
        assert np.array_equal(logits.cpu().numpy(), case.logits), "the input was written"
    assert np.array_equal(got, x32, equal_nan=True), "not the formula's fp32 steps"
    fine = np.isfinite(x64)
    assert np.array_equal(np.isneginf(got), np.isneginf(x64)) and (np.abs(got[fine] - x64[fine]) <= tol[fine]).all()
    chosen = nxt.cpu().numpy()
    assert chosen[case.rows] == -99
    if kw.get("next_", True):
        best = np.where(np.isnan(got), -np.inf, got)
        assert np.array_equal(chosen[:-1], np.where(np.isneginf(best).all(1), -1, best.argmax(1)))
        assert (ws == 0).all(), "the workspace is not zero again"
    else:
        assert (chosen == -99).all()
    return got


@gpu
@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 1000, 4095, 4096, 4097, 32000, 49152, 128257])
def test_logits_vocabularies(torch_mod, dev, vocab):
    check_logits(torch_mod, dev, LogitCase(3, vocab, history=300, biases=9, masks=2, seed=vocab))


@gpu
@pytest.mark.parametrize("history", [0, 1, 255, 257, 5000])
@pytest.mark.parametrize("biases", [0, 1, 400])
@pytest.mark.parametrize("masks", [0, 3])
def test_logits_features(torch_mod, dev, history, biases, masks):
    check_logits(torch_mod, dev, LogitCase(5, 5003, history, biases, masks, seed=history + biases))


@gpu
@pytest.mark.parametrize("rows", [1, 2, 65, 300])
def test_logits_rows(torch_mod, dev, rows):
    check_logits(torch_mod, dev, LogitCase(rows, 9001, 50, 3, min(rows, 7), seed=rows))


@gpu
@pytest.mark.parametrize("rows,vocab,history", [(1, 1, 4097), (2, 40001, 4096), (2, 40001, 4097), (7, 5003, 9000), (8, 9001, 6001), (17, 65001, 4100),
                                                (25, 50257, 5000)])
def test_logits_long_histories(torch_mod, dev, rows, vocab, history):
    check_logits(torch_mod, dev, LogitCase(rows, vocab, history, biases=600, masks=3, seed=rows + history))


@gpu
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("ld,out_ld", [(4100, 4100), (4101, 4101), (4099, 4100), (4100, 5003)])
def test_logits_strides_and_alignment(torch_mod, dev, shift, ld, out_ld):
    case = LogitCase(4, 4099, 60, 5, 2, seed=shift, ld=ld)
    check_logits(torch_mod, dev, case, shift=shift, out_ld=out_ld)
    check_logits(torch_mod, dev, case, shift=shift, in_place=True)


@gpu
def test_logits_options_left_out(torch_mod, dev):
    case = LogitCase(4, 3001, 60, 5, 4, seed=1)
    check_logits(torch_mod, dev, case, next_=False)
    case.mask_of = None  # row r has mask r
    case.prompt_len = None
    check_logits(torch_mod, dev, case)
    case.frequency = None
    check_logits(torch_mod, dev, case)
    case.presence = case.repetition = None
    check_logits(torch_mod, dev, case)


@gpu
def test_logits_odd_values(torch_mod, dev):
    """Tokens outside the vocabulary, lengths outside the stride, infinities and NaN, ties, signed zeros, a mask that leaves nothing."""
    case = LogitCase(6, 5000, 40, 8, 2, seed=2)
    case.history[:, ::5] = -1
    case.history[:, 1::7] = 5000 + 9
    case.history[0, 0], case.history[1, 1] = -2 ** 31, 2 ** 31 - 1
    case.history_len[:] = [40, 41, 1000, -3, 0, 40]
    case.prompt_len[:] = [0, 60, 3, 0, 0, -4]
    case.bias_tokens[:, 3] = case.bias_tokens[:, 1]  # the same token twice: the last value
    case.bias_tokens[:, 4], case.bias_tokens[:, 5] = -1, 5000
    case.bias_len[:] = [8, 9, 2, -1, 0, 8]
    case.mask_of[:] = [-1, -1, 0, 1, -1, -1]
    case.masks[1] = False
    case.logits[0, 10:20] = -np.inf
    case.logits[0, 4000] = np.inf
    case.logits[0, 4500] = np.inf  # a tie: the first
    case.logits[1, 77] = np.nan
    case.logits[4, :] = -1.0
    case.logits[4, 5], case.logits[4, 4999] = -0.0, 0.0
    case.logits[5, :5000] = -np.inf
    case.bias_tokens[5, :] = 100
    x32 = check_logits_any(torch_mod, dev, case)
    assert x32[2][3] == -1 and x32[2][5] == -1 and x32[2][0] == 4000 and x32[2][4] == 5


def check_logits_any(torch, dev, case):
    args, out, nxt, ws, _ = case.call(torch, dev)
    _lib.check(_lib.lib().rh_process_logits(*args, None))
    torch.cuda.synchronize()
    # A prompt length below 0 or past the history is the nearest one that is.
    case.prompt_len = np.clip(case.prompt_len, 0, np.clip(case.history_len, 0, case.history.shape[1]))
    with np.errstate(invalid="ignore"):
        x32, _, _ = case.oracle()
    got = out.cpu().numpy()
    assert np.array_equal(got, x32, equal_nan=True)
    return got, x32, nxt.cpu().numpy()


@gpu
def test_logits_calls_of_other_sizes_share_a_workspace(torch_mod, dev):
    ws = torch_mod.zeros(1 << 20, dtype=torch_mod.uint8, device=dev)
    for rows, vocab in ((3, 50000), (64, 4097), (1, 100), (33, 20000), (3, 50000)):
        check_logits(torch_mod, dev, LogitCase(rows, vocab, 20, 2, 1, seed=rows), workspace=ws)
        check_logits(torch_mod, dev, LogitCase(rows, vocab, 4500, 2, 1, seed=rows), workspace=ws)


@gpu
def test_logits_graph_replays(torch_mod, dev):
    torch = torch_mod
    case = LogitCase(7, 30001, 100, 5, 2, seed=3)
    args, out, nxt, ws, logits = case.call(torch, dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        _lib.check(_lib.lib().rh_process_logits(*args, torch.cuda.current_stream().cuda_stream))
    for _ in range(4):
        logits.copy_(torch.roll(logits, 17, 1))
        out.fill_(0)
        g.replay()
        torch.cuda.synchronize()
        got, chosen = out.clone(), nxt.clone()
        _lib.check(_lib.lib().rh_process_logits(*args, None))
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.equal(chosen, nxt)


# ---- refusals (nothing is launched: the CPU suffices) ------------------------------------------------------

TABLES = dict(cached=16, fresh=16, shared=None, n_seqs=4, group_seqs=None, n_groups=0, block_size=16, tables=16, table_stride=8, free_blocks=16, free_count=16,
              max_rows=4, row_off=16, last_row=16, table_off=16, pos=16, seq=16, slot=16, dec_meta=16, groups=None, totals=16, stream=None)


@pytest.mark.parametrize("change,message", [
    ({"n_seqs": -1}, "bad sizes"), ({"n_groups": -1}, "bad sizes"), ({"block_size": 0}, "bad sizes"), ({"table_stride": 0}, "bad sizes"),
    ({"max_rows": -1}, "bad sizes"), ({"max_rows": 1 << 30}, "2^30"), ({"block_size": 1 << 30}, "2^30"), ({"n_seqs": 1 << 28}, "2^31"),
    ({"cached": None}, "missing"), ({"tables": None}, "missing"), ({"free_count": None}, "missing"), ({"n_groups": 1}, "missing"), ({"slot": None}, "missing"),
    ({"dec_meta": 24}, "aligned"), ({"groups": 8}, "aligned")])
def test_step_tables_refusals(change, message):
    assert _lib.lib().rh_step_tables(*{**TABLES, **change}.values()) != 0
    assert message in _lib.last_error()


QK = dict(qkv=16, planes=1, scale=None, T=4, bias=None, q_norm=16, k_norm=16, eps=1e-6, inv_freq=16, pos=16, slot=16, kpool=16, vpool=16, q_out=16, q_scale=1.0,
          heads=4, kv_heads=2, head_dim=64, block_size=16, stream=None)


@pytest.mark.parametrize("change,message", [
    ({"T": -1}, "bad sizes"), ({"heads": 0}, "bad sizes"), ({"kv_heads": 0}, "bad sizes"), ({"block_size": 0}, "bad sizes"), ({"head_dim": 60}, "head_dim"),
    ({"head_dim": 520}, "head_dim"), ({"head_dim": 0}, "head_dim"), ({"planes": 0}, "planes"), ({"planes": 9}, "planes"), ({"qkv": None}, "missing"),
    ({"q_norm": None}, "missing"), ({"slot": None}, "missing"), ({"q_out": None}, "missing"), ({"qkv": 24}, "aligned"), ({"kpool": 20}, "aligned")])
def test_qk_norm_refusals(change, message):
    assert _lib.lib().rh_qk_norm_to_cache(*{**QK, **change}.values()) != 0
    assert message in _lib.last_error()
    assert _lib.lib().rh_qk_norm_to_cache(*{**QK, "T": 0}.values()) == 0


LOGITS = dict(logits=16, ld=100, rows=2, vocab=100, history=16, history_stride=8, history_len=16, prompt_len=None, repetition=16, frequency=None, presence=None,
              bias_tokens=None, bias_values=None, bias_stride=0, bias_len=None, masks=None, mask_stride=0, mask_of=None, out=32, out_ld=100, next=16,
              workspace=16, workspace_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change,message", [
    ({"rows": -1}, "bad sizes"), ({"vocab": 0}, "bad sizes"), ({"vocab": 1 << 30, "ld": 1 << 30, "out_ld": 1 << 30}, "bad sizes"), ({"ld": 99}, "bad sizes"), ({"out_ld": 99}, "bad sizes"), ({"logits": None}, "missing"),
    ({"out": None}, "missing"), ({"out": 16, "out_ld": 101}, "in place"), ({"history_len": None}, "lengths"), ({"history_stride": -1}, "stride"),
    ({"history": None}, "need a history"), ({"bias_tokens": 16}, "biases need"), ({"bias_tokens": 16, "bias_values": 16, "bias_len": 16, "bias_stride": -1}, "biases need"),
    ({"masks": 16, "mask_stride": 3}, "a bit for each"), ({"workspace": None}, "workspace"), ({"workspace": 20}, "workspace"), ({"workspace_bytes": 8}, "workspace"),
    ({"rows": 1 << 30, "vocab": 100000, "ld": 100000, "out_ld": 100000}, "too many rows")])
def test_logits_refusals(change, message):
    assert _lib.lib().rh_process_logits(*{**LOGITS, **change}.values()) != 0
    assert message in _lib.last_error()
    assert _lib.lib().rh_process_logits(*{**LOGITS, "rows": 0}.values()) == 0
