"""The operators of a decode step together, as a server that keeps its batch on the device runs them:
two groups of requests that share a prompt, decoded greedily under penalties, biases and a
grammar, with metadata, cache writes, attention, logits and the next token on the GPU. The step is
captured once into a graph; every replay is checked against the same step run eagerly, and the
logits against the model in 64 bits on the tokens that were chosen.

Tolerance of the logits: 2e-3 of a row's largest, the bound of this repository's whole-model runs
(fp16 operands, fp32 sums); the model here has two layers.
"""
import math

import numpy as np
import pytest

from relay_amd import _lib

pytestmark = pytest.mark.gpu

H, HEADS, KVH, D, I, V, LAYERS, B = 256, 8, 2, 64, 512, 1003, 2, 16
Q, KV = HEADS * D, KVH * D
EPS = 1e-6
PROMPTS = (50, 32)   # shared tokens of the two groups: 48 of 50 in whole blocks
MEMBERS = 3
N = 2 * MEMBERS
STEPS = 19           # past a block's end
WIDTH, CAP, ROWS = 8, 128, N + 2


class Model:
    def __init__(self, seed):
        r = np.random.default_rng(seed)
        w = lambda *s: (r.standard_normal(s) / math.sqrt(s[-1])).astype(np.float16)  # noqa: E731
        n = lambda k: (1 + 0.1 * r.standard_normal(k)).astype(np.float32)  # noqa: E731
        self.embed, self.head, self.final = (r.standard_normal((V, H))).astype(np.float16), w(V, H), n(H)
        self.layers = [dict(norm=n(H), qkv=w(Q + 2 * KV, H), qn=n(D), kn=n(D), o=w(H, Q), mlp=n(H), gu=w(2 * I, H), down=w(H, I)) for _ in range(LAYERS)]
        self.inv_freq = (10000.0 ** (-np.arange(0, D, 2) / D)).astype(np.float32)

    def logits(self, tokens):
        """Of every position of one sequence, in 64 bits."""
        f = lambda a: a.astype(np.float64)  # noqa: E731
        x = f(self.embed[tokens])
        t = len(tokens)
        angle = np.arange(t)[:, None] * f(self.inv_freq)
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        rms = lambda y, w, eps: y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps) * f(w)  # noqa: E731
        for L in self.layers:
            y = (rms(x, L["norm"], EPS) @ f(L["qkv"]).T).reshape(t, HEADS + 2 * KVH, D)

            def turn(z, w):
                z = rms(z, w, EPS)
                lo, hi = z[..., :D // 2], z[..., D // 2:]
                return np.concatenate([lo * c - hi * s, hi * c + lo * s], -1)

            q, k, v = turn(y[:, :HEADS], L["qn"]), turn(y[:, HEADS:HEADS + KVH], L["kn"]), y[:, HEADS + KVH:]
            out = np.zeros((t, HEADS, D))
            for h in range(HEADS):
                sc = q[:, h] @ k[:, h // (HEADS // KVH)].T / math.sqrt(D)
                sc[np.triu_indices(t, 1)] = -np.inf
                p = np.exp(sc - sc.max(-1, keepdims=True))
                out[:, h] = p / p.sum(-1, keepdims=True) @ v[:, h // (HEADS // KVH)]
            x = x + out.reshape(t, Q) @ f(L["o"]).T
            gu = rms(x, L["mlp"], EPS) @ f(L["gu"]).T
            x = x + (gu[:, :I] / (1 + np.exp(-gu[:, :I])) * gu[:, I:]) @ f(L["down"]).T
        return rms(x, self.final, EPS) @ f(self.head).T


class Server:
    """The device state of the batch and one step over it."""

    def __init__(self, torch, dev, model, seed):
        self.torch, self.lib = torch, _lib.lib()
        r = np.random.default_rng(seed)
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(dev)  # noqa: E731
        i = lambda a: t(np.asarray(a, np.int32))  # noqa: E731
        z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
        self.w = [{k: t(v) for k, v in L.items()} for L in model.layers]
        self.embed, self.head, self.final, self.inv_freq = t(model.embed), t(model.head), t(model.final), t(model.inv_freq)
        blocks = 64
        self.pools = [(z(blocks, KVH, B, D), z(blocks, KVH, B, D)) for _ in range(LAYERS)]
        self.tables, self.free = i(np.full((N, WIDTH), -1)), i(r.permutation(blocks))
        self.totals = i([0, 0, blocks, 0])
        self.cached, self.fresh, self.shared = i(np.zeros(N)), i(np.zeros(N)), i(np.zeros(N))
        self.group_seqs = i([[0, MEMBERS], [MEMBERS, MEMBERS]])
        self.history, self.hist_len, self.prompt_len = i(np.zeros((N, CAP))), i(np.zeros(N)), i(np.zeros(N))
        self.token = i(np.zeros(N))  # of each sequence, the one to decode next
        self.penalties = [t(np.full(N, x, np.float32)) for x in (1.2, 0.3, 0.1)]
        self.bias_tokens, self.bias_values, self.bias_len = i(r.integers(0, V, (N, 5))), t(r.standard_normal((N, 5)).astype(np.float32)), i(np.full(N, 5))
        self.allowed = r.random((1, -(-V // 32) * 32)) < 0.5
        self.masks, self.mask_of = t(np.packbits(self.allowed, axis=1, bitorder="little").view(np.int32)), i([0, -1, -1, 0, -1, -1])
        self.dev, self.z = dev, z
        self.workspaces = {}

    def rows(self, rows):
        """Buffers of a step of up to `rows` rows."""
        z, f, n = self.z, self.torch.float32, self.torch.int32
        return dict(rows=rows, pos=z(rows, dt=n), seq=z(rows, dt=n), slot=z(rows, dt=n), meta=z(rows, 4, dt=n), groups=z(2, 4, dt=n), row_off=z(N + 1, dt=n),
                    last=z(N, dt=n), off=z(N, dt=n), x=z(rows, H, dt=f), xn=z(rows, H), qkv=z(rows, Q + 2 * KV, dt=f), q=z(rows, Q), attn=z(rows, Q),
                    act=z(rows, I), xl=z(N, H), logits=z(N, V, dt=f), out=z(N, V, dt=f), next=z(N, dt=n))

    def workspace(self, size, key):
        if key not in self.workspaces:
            self.workspaces[key] = self.torch.zeros(max(16, size), dtype=self.torch.uint8, device=self.dev)
        return self.workspaces[key]

    def tables_step(self, b, stream):
        p = lambda t: t.data_ptr()  # noqa: E731
        _lib.check(self.lib.rh_step_tables(p(self.cached), p(self.fresh), p(self.shared), N, p(self.group_seqs), 2, B, p(self.tables), WIDTH, p(self.free),
                                           p(self.totals) + 8, b["rows"], p(b["row_off"]), p(b["last"]), p(b["off"]), p(b["pos"]), p(b["seq"]), p(b["slot"]),
                                           p(b["meta"]), p(b["groups"]), p(self.totals), stream), "step tables")

    def forward(self, b, tokens, stream):
        L, p, T = self.lib, lambda t: t.data_ptr(), b["rows"]
        n_groups, members, shared, own = 2, MEMBERS, max(PROMPTS), CAP
        size = L.rh_shared_prefix_workspace(T, n_groups, members, shared, own, HEADS, KVH, D)
        ws = self.workspace(size, "attention %d" % T)
        ok = _lib.check
        gemv = lambda w, x, y, k, n, beta: [ok(L.rh_gemv_f16(p(w), k, x.data_ptr() + 2 * k * r0, y.data_ptr() + 4 * n * r0, min(32, T - r0), k, n, beta, stream))  # noqa: E731
                                            for r0 in range(0, T, 32)]
        ok(L.rh_embed(p(tokens), T, p(self.embed), H, p(b["x"]), stream))
        for w, (kp, vp) in zip(self.w, self.pools):
            ok(L.rh_rmsnorm(p(b["x"]), None, T, p(w["norm"]), H, EPS, p(b["xn"]), stream))
            gemv(w["qkv"], b["xn"], b["qkv"], H, Q + 2 * KV, 0.0)
            ok(L.rh_qk_norm_to_cache(p(b["qkv"]), 1, None, T, None, p(w["qn"]), p(w["kn"]), EPS, p(self.inv_freq), p(b["pos"]), p(b["slot"]), p(kp), p(vp),
                                     p(b["q"]), 1.0, HEADS, KVH, D, B, stream))
            ok(L.rh_shared_prefix_attention(p(b["q"]), Q, p(kp), p(vp), p(b["meta"]), p(b["groups"]), p(self.tables), T, n_groups, members, shared, own,
                                            HEADS, KVH, D, B, 1 / math.sqrt(D), p(ws), ws.numel(), p(b["attn"]), Q, stream))
            gemv(w["o"], b["attn"], b["x"], Q, H, 1.0)
            ok(L.rh_rmsnorm(p(b["x"]), None, T, p(w["mlp"]), H, EPS, p(b["xn"]), stream))
            for r0 in range(0, T, 32):
                ok(L.rh_gemv_f16_gate_up_silu(p(w["gu"]), H, p(b["xn"]) + 2 * H * r0, p(b["act"]) + 2 * I * r0, min(32, T - r0), H, I, stream))
            gemv(w["down"], b["act"], b["x"], I, H, 1.0)
        ok(L.rh_rmsnorm(p(b["x"]), p(b["last"]), N, p(self.final), H, EPS, p(b["xl"]), stream))
        ok(L.rh_gemv_f16(p(self.head), H, p(b["xl"]), p(b["logits"]), N, H, V, 0.0, stream))

    def choose(self, b, stream):
        L, p = self.lib, lambda t: t.data_ptr()  # noqa: E731
        size = L.rh_process_logits_workspace(N, V)
        ws = self.workspace(size, "logits")
        _lib.check(L.rh_process_logits(p(b["logits"]), V, N, V, p(self.history), CAP, p(self.hist_len), p(self.prompt_len), *map(p, self.penalties),
                                       p(self.bias_tokens), p(self.bias_values), 5, p(self.bias_len), p(self.masks), self.masks.shape[1], p(self.mask_of),
                                       p(b["out"]), V, p(b["next"]), p(ws), ws.numel(), stream), "logits")

    def decode(self, b, stream):
        """One token of every sequence: metadata, model, token, and the state behind it."""
        self.tables_step(b, stream)
        self.forward(b, self.token.index_select(0, b["seq"]), stream)
        self.choose(b, stream)
        self.token.copy_(b["next"])
        self.history.scatter_(1, self.hist_len.long()[:, None], b["next"][:, None])
        self.hist_len.add_(1)
        self.cached.add_(self.fresh)

    STATE = ("tables", "totals", "cached", "history", "hist_len", "token")

    def state(self):
        return [getattr(self, k).clone() for k in self.STATE] + [t.clone() for kv in self.pools for t in kv]

    def restore(self, state):
        for t, s in zip([getattr(self, k) for k in self.STATE] + [t for kv in self.pools for t in kv], state):
            t.copy_(s)


def admit(torch, server, prompts, stream):
    """The groups' prompts: the first member of each computes its own, a step of many rows; the others take its whole blocks and compute the rest."""
    tail = []
    for first, prompt in zip((0, MEMBERS), prompts):
        server.fresh.zero_()
        server.fresh[first] = len(prompt)
        b = server.rows(len(prompt) + 3)
        server.tables_step(b, stream)
        tokens = torch.zeros(b["rows"], dtype=torch.int32, device=server.dev)
        tokens[:len(prompt)] = torch.tensor(prompt, dtype=torch.int32, device=server.dev)
        server.forward(b, tokens, stream)
        server.cached[first] = len(prompt)
        tail.append(b["logits"][first].double().cpu().numpy())
    for first, prompt in zip((0, MEMBERS), prompts):
        whole = len(prompt) // B
        for s in range(first + 1, first + MEMBERS):
            server.tables[s, :whole] = server.tables[first, :whole]
            server.cached[s] = whole * B
        server.shared[first:first + MEMBERS] = whole * B
        rest = len(prompt) - whole * B
        if rest:  # the tokens behind the last whole block, by every other member itself
            server.fresh.zero_()
            server.fresh[first + 1:first + MEMBERS] = rest
            b = server.rows(rest * (MEMBERS - 1))
            server.tables_step(b, stream)
            server.forward(b, torch.tensor(prompt[whole * B:] * (MEMBERS - 1), dtype=torch.int32, device=server.dev), stream)
            server.cached.add_(server.fresh)
    server.fresh.fill_(1)
    return tail


def test_decode_loop_on_the_device(torch_mod, dev):
    torch = torch_mod
    model = Model(1)
    r = np.random.default_rng(2)
    prompts = [[int(x) for x in r.integers(0, V, n)] for n in PROMPTS]
    server = Server(torch, dev, model, 3)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        tail = admit(torch, server, prompts, stream.cuda_stream)
        for s in range(N):
            prompt = prompts[s // MEMBERS]
            server.history[s, :len(prompt)] = torch.tensor(prompt, dtype=torch.int32, device=dev)
            server.hist_len[s], server.prompt_len[s] = len(prompt), len(prompt)
            server.token[s] = 7 * s + 1  # the members go different ways
        stream.synchronize()
        for got, prompt in zip(tail, prompts):
            want = model.logits(prompt)[-1]
            assert np.abs(got - want).max() <= 2e-3 * np.abs(want).max()
        server.history.scatter_(1, server.hist_len.long()[:, None], server.token[:, None])
        server.hist_len.add_(1)
        b = server.rows(ROWS)
        before = server.state()
        server.decode(b, stream.cuda_stream)  # the first run outside the graph
        server.restore(before)
        stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        server.decode(b, torch.cuda.current_stream().cuda_stream)
    chosen, logits = [server.token.cpu().numpy().copy()], []
    eager = server.rows(ROWS)
    for step in range(STEPS):
        before = server.state()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        after = server.state()
        server.restore(before)
        server.decode(eager, None)
        torch.cuda.synchronize()
        for k, (x, y) in enumerate(zip(after, server.state())):
            assert torch.equal(x, y), f"step {step}: state {k} of the replay is not the eager one"
        for k in ("logits", "out", "next", "slot", "meta", "groups"):
            assert torch.equal(b[k], eager[k]), f"step {step}: {k}"
        assert server.totals.tolist()[0] == N and server.totals.tolist()[3] == 0
        chosen.append(server.token.cpu().numpy().copy())
        logits.append(b["logits"].double().cpu().numpy())
        out = b["out"].cpu().numpy()
        assert np.isneginf(out[[0, 3]][:, ~server.allowed[0, :V]]).all() and np.array_equal(chosen[-1], out.argmax(1))
    # The members' tables share their prompts' whole blocks, nothing else, and no block twice.
    tables = server.tables.cpu().numpy()
    held = [tables[s, :-(-int(c) // B)].tolist() for s, c in enumerate(server.cached.cpu())]
    for first, prompt in zip((0, MEMBERS), prompts):
        whole = len(prompt) // B
        assert all(held[s][:whole] == held[first][:whole] for s in range(first, first + MEMBERS))
    every = [x for s, h in enumerate(held) for x in (h if s % MEMBERS == 0 else h[len(prompts[s // MEMBERS]) // B:])]
    assert len(set(every)) == len(every) and server.totals.tolist()[2] == 64 - len(every)
    for s in range(N):
        prompt = prompts[s // MEMBERS]
        want = model.logits(prompt + [int(c[s]) for c in chosen[:-1]])[len(prompt):]
        for step in range(STEPS):
            off = np.abs(logits[step][s] - want[step]).max() / np.abs(want[step]).max()
            assert off <= 2e-3, f"sequence {s}, step {step}: off by {off}"
