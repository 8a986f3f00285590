"""The operators of a decode step that stays on the GPU, as cases to time and check.

A server that keeps its batch on the device runs four operators around the products of a
layer: block tables and slot maps of the step from the request lengths (`rh_step_tables`), the
norm of queries and keys per head with the rotation and the cache write (`rh_qk_norm_to_cache`),
attention of sequences that share a prompt (`rh_shared_prefix_attention`), and penalties, biases and
grammar masks on the logits with the greedy token (`rh_process_logits`).

`run` computes each in its plain form from elementary torch operations, or, with `own` set,
through the library's calls. Head counts are those of the three models that the benchmark runs
(9/3 heads of 64, 32/4 of 64, 32/8 of 128) and a few generic ones.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
EPS = 1e-6


def listed():
    return [
        # Two requests on one short system prompt: the smallest attention call, latency only.
        {"name": "shared_2x512_9_3_64", "kind": "shared", "groups": 1, "members": 2, "shared": 512, "own": 40, "heads": 9, "kv_heads": 3,
         "dim": 64, "block": 16},
        # A chat service: 32 conversations on one long system prompt.
        {"name": "shared_32x2048_32_4_64", "kind": "shared", "groups": 1, "members": 32, "shared": 2048, "own": 300, "heads": 32, "kv_heads": 4,
         "dim": 64, "block": 16},
        # Parallel samples: five prompts, each answered nine times, in blocks of 32.
        {"name": "shared_5x9x1504_32_8_128", "kind": "shared", "groups": 5, "members": 9, "shared": 1504, "own": 700, "heads": 32, "kv_heads": 8,
         "dim": 128, "block": 32},
        # 64 requests about one long document: the largest call.
        {"name": "shared_64x16384_32_8_128", "kind": "shared", "groups": 1, "members": 64, "shared": 16384, "own": 1000, "heads": 32,
         "kv_heads": 8, "dim": 128, "block": 16},
        # The metadata of one decode step of 48 sequences.
        {"name": "tables_48_decode", "kind": "tables", "seqs": 48, "chunk": 1, "chunks": 0, "context": 8192, "groups": 2, "block": 16},
        # A step that admits 40 prompts of up to 701 tokens beside 471 decoding sequences.
        {"name": "tables_511_mixed", "kind": "tables", "seqs": 511, "chunk": 701, "chunks": 40, "context": 4096, "groups": 16, "block": 16},
        # One token of one user.
        {"name": "qk_norm_1_9_3_64", "kind": "qk_norm", "tokens": 1, "heads": 9, "kv_heads": 3, "dim": 64, "planes": 1, "bias": False},
        # A decode batch whose projection left three K ranges to add.
        {"name": "qk_norm_48_32_8_128_p3", "kind": "qk_norm", "tokens": 48, "heads": 32, "kv_heads": 8, "dim": 128, "planes": 3, "bias": True},
        # A whole prompt in one chunk.
        {"name": "qk_norm_2047_32_4_64", "kind": "qk_norm", "tokens": 2047, "heads": 32, "kv_heads": 4, "dim": 64, "planes": 1, "bias": False},
        # One user with a repetition penalty over a small vocabulary.
        {"name": "logits_1x49152", "kind": "logits", "rows": 1, "vocab": 49152, "history": 640, "biases": 0, "masks": 0},
        # A decode batch, half of it under JSON grammars.
        {"name": "logits_48x32000_masks", "kind": "logits", "rows": 48, "vocab": 32000, "history": 2048, "biases": 20, "masks": 24},
        # A large batch over a large, odd vocabulary with long histories.
        {"name": "logits_64x128257", "kind": "logits", "rows": 64, "vocab": 128257, "history": 8000, "biases": 300, "masks": 16},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "tables", "qk_norm", "logits"])
    heads, kv_heads, dim = rng.choice([(9, 3, 64), (32, 4, 64), (32, 8, 128), (14, 2, 64), (8, 8, 32), (16, 1, 128)])
    if kind == "shared":
        groups, block = _log_int(rng, 1, 6), rng.choice([16, 16, 32, 64])
        return {"kind": kind, "groups": groups, "members": _log_int(rng, 1, 60 // groups), "shared": block * _log_int(rng, 1, 14000 // block),
                "own": _log_int(rng, 1, 1000), "heads": heads, "kv_heads": kv_heads, "dim": dim, "block": block}
    if kind == "tables":
        seqs = _log_int(rng, 1, 511)
        return {"kind": kind, "seqs": seqs, "chunk": _log_int(rng, 2, 701), "chunks": min(seqs, rng.choice([0, _log_int(rng, 1, 40)])),
                "context": _log_int(rng, 16, 8192), "groups": min(seqs, rng.choice([0, 1, 7])), "block": rng.choice([16, 16, 32, 12])}
    if kind == "qk_norm":
        return {"kind": kind, "tokens": _log_int(rng, 1, 4096), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "planes": rng.choice([1, 1, 2, 3]), "bias": rng.random() < 0.5}
    rows = _log_int(rng, 1, 64)
    return {"kind": kind, "rows": rows, "vocab": _log_int(rng, 1000, 128257), "history": _log_int(rng, 1, 8000),
            "biases": rng.choice([0, _log_int(rng, 1, 300)]), "masks": rng.choice([0, _log_int(rng, 1, rows)])}


# ---- inputs from a seed ----------------------------------------------------------------------------

def _gen(seed, salt=0):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1000003 + salt)


def _ints(values):
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).to(DEV)


def prepare(case, seed):
    return globals()["_prepare_" + case["kind"]](case, seed)


def run(state):
    return globals()[("_own_" if own else "_plain_") + state["case"]["kind"]](state)


def work(case):
    return globals()["_work_" + case["kind"]](case)


def exact(case, seed):
    return globals()["_exact_" + case["kind"]](prepare(case, seed))


def _own_call(state, name, build):
    """The bound call of a state, on the current stream: a program that decodes step after step keeps its argument list, workspaces and
    output buffers (so the next run writes what this one returned) and looks up no more than its stream."""
    if "call" not in state:
        from relay_amd import _lib
        fn, args, check = getattr(_lib.lib(), name), build(_lib.lib()), _lib.check
        stream, device = torch._C._cuda_getCurrentRawStream, torch.cuda.current_device()

        def call():
            check(fn(*args, stream(device)), name)
        state["call"] = call
    state["call"]()


def _p(t):
    return 0 if t is None else t.data_ptr()


# ---- attention over a shared prefix ---------------------------------------------------------------

def _own_lengths(case, seed):
    return np.random.default_rng(seed + 29).integers(max(1, case["own"] // 4), case["own"] + 1, size=case["groups"] * case["members"])


def _prepare_shared(case, seed):
    r = np.random.default_rng(seed)
    ng, m, p, b = case["groups"], case["members"], case["shared"], case["block"]
    heads, kvh, d = case["heads"], case["kv_heads"], case["dim"]
    own_keys = _own_lengths(case, seed)
    n, sb = ng * m, p // b
    ob = -(-own_keys // b)
    nb = int(ng * sb + ob.sum())
    ids = r.permutation(nb)
    width = int(sb + ob.max())
    tables = np.zeros((n, width), np.int32)
    at = ng * sb
    for i in range(n):
        g = i // m
        tables[i, :sb] = ids[g * sb:(g + 1) * sb]
        tables[i, sb:sb + ob[i]] = ids[at:at + ob[i]]
        at += int(ob[i])
    rows = r.permutation(n)  # descriptors are ordered by group, rows of q by request
    meta = np.stack([rows, p + own_keys, np.arange(n) * width, np.full(n, p)], 1)
    groups = np.stack([np.arange(ng) * m, np.full(ng, m), np.full(ng, p), np.arange(ng) * m * width], 1)
    g = _gen(seed, 1)
    return {"case": case, "max_own": case["own"], "k": torch.randn(nb, kvh, b, d, generator=g, device=DEV, dtype=torch.float16),
            "v": torch.randn(nb, kvh, b, d, generator=g, device=DEV, dtype=torch.float16),
            "q": (torch.randn(n, heads * d, generator=g, device=DEV) * 1.5).half(), "meta": _ints(meta), "groups": _ints(groups),
            "tables": _ints(tables), "out": torch.empty(n, heads * d, device=DEV, dtype=torch.float16)}


def _plain_shared(s):
    c = s["case"]
    heads, kvh, d, b = c["heads"], c["kv_heads"], c["dim"], c["block"]
    n, width = s["tables"].shape
    grp = heads // kvh
    row, ctx = s["meta"][:, 0].long(), s["meta"][:, 1]
    at = s["tables"].long()
    k = s["k"][at].float().permute(0, 2, 4, 1, 3).reshape(n * kvh, d, width * b)
    v = s["v"][at].float().permute(0, 2, 1, 3, 4).reshape(n * kvh, width * b, d)
    q = s["q"][row].float().reshape(n * kvh, grp, d)
    scores = torch.bmm(q, k).reshape(n, kvh * grp, width * b) / math.sqrt(d)
    seen = torch.arange(width * b, device=DEV)[None, None, :] < ctx[:, None, None]
    scores = torch.where(seen, scores, float("-inf"))
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    w = e / e.sum(-1, keepdim=True)
    o = torch.bmm(w.reshape(n * kvh, grp, width * b), v).reshape(n, heads * d)
    out = torch.empty_like(s["out"])
    out[row] = o.half()
    return out


def _own_shared(s):
    def build(lib):
        c = s["case"]
        n, ng = s["meta"].shape[0], s["groups"].shape[0]
        heads, kvh, d = c["heads"], c["kv_heads"], c["dim"]
        size = lib.rh_shared_prefix_workspace(n, ng, c["members"], c["shared"], s["max_own"], heads, kvh, d)
        s["workspace"] = torch.zeros(max(1, size), dtype=torch.uint8, device=DEV)
        return (_p(s["q"]), heads * d, _p(s["k"]), _p(s["v"]), _p(s["meta"]), _p(s["groups"]), _p(s["tables"]), n, ng, c["members"],
                c["shared"], s["max_own"], heads, kvh, d, c["block"], 1.0 / math.sqrt(d), _p(s["workspace"]), size, _p(s["out"]), heads * d)
    _own_call(s, "rh_shared_prefix_attention", build)
    return s["out"]


def _exact_shared(s):
    c = s["case"]
    heads, kvh, d, b = c["heads"], c["kv_heads"], c["dim"], c["block"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    tables = s["tables"].long()

    def rows_of(pool, blocks):  # [kv heads][keys][dim]
        return pool[blocks].double().transpose(0, 1).reshape(kvh, -1, d)

    for i, (row, ctx, _, shared) in enumerate(s["meta"].tolist()):
        blocks = tables[i, :-(-ctx // b)]
        q = s["q"][row].double().reshape(kvh, heads // kvh, d)
        logit = q @ rows_of(s["k"], blocks)[:, :ctx].transpose(1, 2) * d ** -0.5
        out[row] = (torch.softmax(logit, -1) @ rows_of(s["v"], blocks)[:, :ctx]).reshape(-1)
    return out


def _work_shared(case):
    n = case["groups"] * case["members"]
    mean_own = (max(1, case["own"] // 4) + case["own"]) / 2
    keys = case["groups"] * case["shared"] + n * mean_own
    return {"bytes": 4 * keys * case["kv_heads"] * case["dim"] + 4 * n * case["heads"] * case["dim"],
            "flops": 4 * n * case["heads"] * case["dim"] * (case["shared"] + mean_own)}


# ---- block tables and slot maps --------------------------------------------------------------------

def _lengths(case, seed):
    r = np.random.default_rng(seed + 3)
    n = case["seqs"]
    cached = r.integers(0, case["context"] + 1, size=n)
    fresh = np.ones(n, np.int64)
    pick = r.permutation(n)[:case["chunks"]]
    fresh[pick] = r.integers(-(-3 * case["chunk"] // 4), case["chunk"] + 1, size=len(pick))
    fresh[r.random(n) < 0.05] = 0  # requests that wait this step
    return cached, fresh


def _budget(case):
    """Rows of the step's buffers: what the step may hold at most; those past its tokens stay idle."""
    return case["seqs"] + case["chunks"] * (case["chunk"] - 1)


def _prepare_tables(case, seed):
    r = np.random.default_rng(seed)
    n, b, ng = case["seqs"], case["block"], case["groups"]
    cached, fresh = _lengths(case, seed)
    held, want = -(-cached // b), -(-(cached + fresh) // b)
    width = -(-(case["context"] + case["chunk"]) // b) + 1
    total = int(held.sum() + (want - held).sum()) + 64
    ids = r.permutation(total)
    start = np.concatenate([[0], np.cumsum(held)])
    tables = np.full((n, width), -1, np.int32)
    for i in range(n):
        tables[i, :held[i]] = ids[start[i]:start[i + 1]]
    free = ids[start[-1]:]
    bounds = np.linspace(0, n, ng + 1).astype(int) if ng else np.zeros(1, int)
    groups = np.stack([bounds[:-1], np.diff(bounds)], 1) if ng else np.zeros((0, 2), int)
    shared = np.zeros(n, int)
    for lo, hi in zip(bounds[:-1], bounds[1:]):
        shared[lo:hi] = cached[lo:hi].min() // b * b if hi > lo else 0
    rows = _budget(case)
    e = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"case": case, "cached": _ints(cached), "fresh": _ints(fresh), "shared": _ints(shared), "group_seqs": _ints(groups), "tables": _ints(tables),
            "free": _ints(free), "free_count": _ints([len(free)]), "rows": rows, "row_off": e(n + 1), "last_row": e(n), "table_off": e(n), "pos": e(rows),
            "seq": e(rows), "slot": e(rows), "meta": e(rows, 4), "groups": e(max(1, ng), 4), "totals": e(4)}


def _tables_outputs(s):
    return {k: s[k] for k in ("tables", "row_off", "last_row", "table_off", "pos", "seq", "slot", "meta", "groups", "totals")}


def _plain_tables(s):
    c = s["case"]
    b, n, ng, rows = c["block"], c["seqs"], c["groups"], s["rows"]
    cached, fresh = s["cached"].long(), s["fresh"].long()
    width = s["tables"].shape[1]
    held, want = (cached + b - 1) // b, (cached + fresh + b - 1) // b
    zero = torch.zeros(1, dtype=torch.long, device=DEV)
    row_off = torch.cat([zero, torch.cumsum(fresh, 0)])
    taken = torch.cat([zero, torch.cumsum(want - held, 0)])
    col = torch.arange(width, device=DEV)[None, :]
    is_new = (col >= held[:, None]) & (col < want[:, None])
    nth = s["free_count"].long() - 1 - (taken[:-1, None] + col - held[:, None])
    tables = torch.where(is_new, s["free"][nth.clamp(0, s["free"].numel() - 1)], s["tables"])
    t = torch.arange(rows, device=DEV)
    live = t < row_off[-1]
    seq = (torch.searchsorted(row_off, t, right=True) - 1).clamp(0, n - 1)
    pos = cached[seq] + t - row_off[seq]
    block = tables[seq, (pos // b).clamp(0, width - 1)].long()
    table_off = torch.arange(n, device=DEV) * width
    off = lambda x, idle: torch.where(live, x, idle)  # noqa: E731
    meta = torch.stack([t, off(pos + 1, 0), off(table_off[seq], 0), off(s["shared"].long()[seq], 0)], 1)
    first = s["group_seqs"][:, 0].long()
    members = row_off[first + s["group_seqs"][:, 1]] - row_off[first]
    groups = torch.stack([row_off[first], members, s["shared"].long()[first], first * width], 1) if ng else torch.zeros(1, 4, device=DEV)
    totals = torch.stack([row_off[-1], taken[-1], s["free_count"][0].long() - taken[-1], zero[0]])
    i = lambda x: x.to(torch.int32)  # noqa: E731
    return {"tables": tables, "row_off": i(row_off), "last_row": i(torch.where(fresh > 0, row_off[1:] - 1, 0)), "table_off": i(table_off),
            "pos": i(off(pos, 0)), "seq": i(off(seq, 0)), "slot": i(off(block * b + pos % b, -1)), "meta": i(meta), "groups": i(groups), "totals": i(totals)}


def _own_tables(s):
    def build(lib):
        c = s["case"]
        return (_p(s["cached"]), _p(s["fresh"]), _p(s["shared"]), c["seqs"], _p(s["group_seqs"]) if c["groups"] else 0, c["groups"], c["block"],
                _p(s["tables"]), s["tables"].shape[1], _p(s["free"]), _p(s["free_count"]), s["rows"], _p(s["row_off"]), _p(s["last_row"]),
                _p(s["table_off"]), _p(s["pos"]), _p(s["seq"]), _p(s["slot"]), _p(s["meta"]), _p(s["groups"]), _p(s["totals"]))
    _own_call(s, "rh_step_tables", build)
    return _tables_outputs(s)


def _exact_tables(s):
    return None  # whole numbers throughout


def _work_tables(case):
    rows = case["seqs"] * 0.95 + case["chunks"] * (case["chunk"] - 1) * 0.83
    new = rows / case["block"]
    return {"bytes": 12 * case["seqs"] + 8 * new + 4 * rows + 28 * _budget(case) + 12 * case["seqs"] + 24 * case["groups"], "flops": 0}


# ---- norm of q and k per head, rotation, cache write ------------------------------------------------

def _prepare_qk_norm(case, seed):
    t, heads, kvh, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    b, width = 16, (heads + 2 * kvh) * d
    r = np.random.default_rng(seed)
    nb = -(-t // b) + 4
    g = _gen(seed, 5)
    inv_freq = 500000.0 ** (-np.arange(0, d, 2, dtype=np.float64) / d)
    pool = lambda: torch.randn(nb, kvh, b, d, generator=g, device=DEV, dtype=torch.float16)  # noqa: E731
    qkv = torch.randn(case["planes"], t, width, generator=g, device=DEV)
    qkv *= torch.rand(width, generator=g, device=DEV) * 3 + 0.1  # channels of different size
    return {"case": case, "block": b, "qkv": qkv, "bias": torch.randn(width, generator=g, device=DEV) if case["bias"] else None,
            "q_norm": 1 + 0.2 * torch.randn(d, generator=g, device=DEV), "k_norm": 1 + 0.2 * torch.randn(d, generator=g, device=DEV),
            "inv_freq": torch.from_numpy(inv_freq.astype(np.float32)).to(DEV), "pos": _ints(r.integers(0, 131072, size=t)),
            "slot": _ints(r.permutation(nb * b)[:t]), "k": pool(), "v": pool(), "q_scale": 1.4426950408889634 / math.sqrt(d),
            "q": torch.zeros(t, heads * d, device=DEV, dtype=torch.float16)}


def _plain_qk_norm(s):
    c = s["case"]
    t, heads, kvh, d, b = c["tokens"], c["heads"], c["kv_heads"], c["dim"], s["block"]
    x = s["qkv"].sum(0)
    if s["bias"] is not None:
        x = x + s["bias"]
    x = x.reshape(t, heads + 2 * kvh, d)
    qk = x[:, :heads + kvh]
    w = torch.cat([s["q_norm"].expand(heads, d), s["k_norm"].expand(kvh, d)])
    qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    angle = s["pos"].double()[:, None] * s["inv_freq"].double()[None, :]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    lo, hi = qk[..., :d // 2], qk[..., d // 2:]
    qk = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    block, at = s["slot"].long() // b, s["slot"].long() % b
    s["k"][block, :, at] = qk[:, heads:].half()
    s["v"][block, :, at] = x[:, heads + kvh:].half()
    return {"q": (qk[:, :heads] * s["q_scale"]).reshape(t, heads * d).half(), "k": s["k"], "v": s["v"]}


def _own_qk_norm(s):
    def build(lib):
        c = s["case"]
        return (_p(s["qkv"]), c["planes"], 0, c["tokens"], _p(s["bias"]), _p(s["q_norm"]), _p(s["k_norm"]), EPS, _p(s["inv_freq"]), _p(s["pos"]),
                _p(s["slot"]), _p(s["k"]), _p(s["v"]), _p(s["q"]), s["q_scale"], c["heads"], c["kv_heads"], c["dim"], s["block"])
    _own_call(s, "rh_qk_norm_to_cache", build)
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _exact_qk_norm(s):
    c = s["case"]
    heads, kvh, d, b = c["heads"], c["kv_heads"], c["dim"], s["block"]
    x = s["qkv"].double().sum(0) + (0 if s["bias"] is None else s["bias"].double())
    q, k, v = x.split([heads * d, kvh * d, kvh * d], 1)
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV), s["pos"].double()[:, None, None] * s["inv_freq"].double())

    def rotated(y, weight):
        y = y.unflatten(1, (-1, d))
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * weight.double()
        z = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    pools = [s["k"].double(), s["v"].double()]
    for pool, rows in zip(pools, (rotated(k, s["k_norm"]), v.unflatten(1, (-1, d)))):
        flat = pool.transpose(1, 2).contiguous()
        flat.view(-1, kvh, d)[s["slot"].long()] = rows
        pool.copy_(flat.transpose(1, 2))
    return {"q": (rotated(q, s["q_norm"]) * s["q_scale"]).flatten(1), "k": pools[0], "v": pools[1]}


def _work_qk_norm(case):
    values = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    return {"bytes": values * (4 * case["planes"] + 2) + 8 * case["tokens"], "flops": 10 * values}


# ---- penalties, biases and masks on logits ----------------------------------------------------------

def _prepare_logits(case, seed):
    r, v, h = case["rows"], case["vocab"], case["history"]
    g, np_r = _gen(seed, 9), np.random.default_rng(seed)
    u = torch.rand(r, h, generator=g, device=DEV)
    history = (v * u ** 4).to(torch.int32).clamp(max=v - 1)  # common tokens come often
    length = np_r.integers(h // 2 + h % 2, h + 1, size=r)
    prompt = (length * np_r.random(r)).astype(np.int64)
    params = torch.rand(3, r, generator=g, device=DEV)
    nbias, nm = case["biases"], case["masks"]
    mask_of = np.full(r, -1)
    mask_of[np_r.permutation(r)[:nm]] = np.arange(nm)
    words = -(-v // 32)
    bits = lambda: torch.randint(-2 ** 31, 2 ** 31, (max(1, nm), words), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)  # noqa: E731
    return {"case": case, "logits": torch.randn(r, v, generator=g, device=DEV) * 4, "history": history, "history_len": _ints(length),
            "prompt_len": _ints(prompt), "repetition": 1 + 0.3 * params[0], "frequency": 0.5 * params[1], "presence": params[2] - 0.2,
            "bias_tokens": torch.randint(0, v, (r, max(1, nbias)), generator=g, device=DEV, dtype=torch.int32),
            "bias_values": torch.randn(r, max(1, nbias), generator=g, device=DEV) * 3, "bias_len": _ints(np.full(r, nbias)),
            "masks": bits() & bits() & bits(), "mask_of": _ints(mask_of),  # a grammar lets an eighth through
            "out": torch.empty(r, v, device=DEV), "next": torch.empty(r, dtype=torch.int32, device=DEV)}


def _plain_logits(s):
    c = s["case"]
    r, v, h = c["rows"], c["vocab"], c["history"]
    at = torch.arange(h, device=DEV)[None, :]
    held, prompt = at < s["history_len"][:, None], at < s["prompt_len"][:, None]
    tokens = s["history"].long()
    zeros = torch.zeros(r, v, dtype=torch.int32, device=DEV)
    seen = zeros.scatter_add(1, tokens, held.int())
    count = zeros.scatter_add(1, tokens, (held & ~prompt).int()).float()
    x, rep = s["logits"], s["repetition"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - torch.where(count > 0, s["presence"][:, None], 0.0)
    if c["biases"]:  # a token named twice has the last of its values
        n = torch.arange(1, c["biases"] + 1, device=DEV, dtype=torch.int32).expand(r, -1).contiguous()
        last = zeros.scatter_reduce(1, s["bias_tokens"].long(), n, "amax").long()
        x = x + torch.where(last > 0, torch.gather(s["bias_values"], 1, (last - 1).clamp(min=0)), 0.0)
    if c["masks"]:
        token = torch.arange(v, device=DEV)
        allowed = (s["masks"][:, token // 32] >> (token % 32).int()) & 1
        of = s["mask_of"].long()
        x = torch.where((of[:, None] < 0) | (allowed[of.clamp(min=0)] > 0), x, float("-inf"))
    return {"out": x, "next": torch.argmax(x, 1).int()}


def _own_logits(s):
    def build(lib):
        c = s["case"]
        r, v = c["rows"], c["vocab"]
        size = lib.rh_process_logits_workspace(r, v)
        s["workspace"] = torch.zeros(max(1, size), dtype=torch.uint8, device=DEV)
        bias, mask = c["biases"] > 0, c["masks"] > 0
        return (_p(s["logits"]), v, r, v, _p(s["history"]), c["history"], _p(s["history_len"]), _p(s["prompt_len"]), _p(s["repetition"]),
                _p(s["frequency"]), _p(s["presence"]), _p(s["bias_tokens"]) if bias else 0, _p(s["bias_values"]) if bias else 0, c["biases"],
                _p(s["bias_len"]) if bias else 0, _p(s["masks"]) if mask else 0, s["masks"].shape[1], _p(s["mask_of"]) if mask else 0,
                _p(s["out"]), v, _p(s["next"]), _p(s["workspace"]), size)
    _own_call(s, "rh_process_logits", build)
    return {"out": s["out"], "next": s["next"]}


def _exact_logits(s):
    c = s["case"]
    x = s["logits"].double().cpu().numpy()
    host = {k: s[k].cpu().numpy() for k in ("history", "history_len", "prompt_len", "repetition", "frequency", "presence", "bias_tokens", "bias_values",
                                            "masks", "mask_of")}
    for r in range(c["rows"]):
        said = host["history"][r, :host["history_len"][r]]
        for token in np.unique(said):
            x[r, token] = x[r, token] / host["repetition"][r].astype(float) if x[r, token] > 0 else x[r, token] * host["repetition"][r].astype(float)
        token, times = np.unique(said[host["prompt_len"][r]:], return_counts=True)
        x[r, token] -= host["frequency"][r].astype(float) * times + host["presence"][r].astype(float)
        named = dict(zip(host["bias_tokens"][r, :c["biases"]].tolist(), host["bias_values"][r, :c["biases"]].tolist()))
        for token, value in named.items():
            x[r, token] += value
        if c["masks"] and host["mask_of"][r] >= 0:
            bits = np.unpackbits(host["masks"][host["mask_of"][r]].view(np.uint8), bitorder="little")[:c["vocab"]]
            x[r, bits == 0] = -np.inf
    return {"out": x, "next": None}


def _work_logits(case):
    r, v = case["rows"], case["vocab"]
    return {"bytes": 8 * r * v + case["masks"] * v / 8 + 0.75 * 4 * r * case["history"] + 8 * r * case["biases"] + 24 * r, "flops": 2 * r * v}
