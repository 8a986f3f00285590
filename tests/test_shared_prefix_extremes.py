"""rh_shared_prefix_attention where fp32 scores or fp16 weights come to their ends."""
import math

import numpy as np
import pytest

from helpers import bits_to_f32, f16_bits
from relay_amd import _lib
from test_shared_prefix import Call, Case

gpu = pytest.mark.gpu


def run(torch, dev, case, tol_of, **kw):
    """The call against attention in 64 bits; tol_of(o, w|v|, keys, max|v|, score size) is a value's tolerance."""
    print(f"shared prefix: groups={[(g[1], g[2]) for g in case.groups][:6]} n={case.n} {case.heads}/{case.kv_heads} D={case.D} bs={case.bs} {kw}", flush=True)
    call = Call(torch, dev, case, **kw)
    call()
    torch.cuda.synchronize()
    got = call.out.cpu().numpy().astype(np.float64)
    q, k, v = (bits_to_f32(x).astype(np.float64) for x in (case.q, case.k, case.v))
    G, D = case.heads // case.kv_heads, case.D
    for (row, c, _, _), where in zip(case.meta, case.keys):
        b, s = (np.array(x) for x in zip(*where))
        for h in range(case.heads):
            K, V, x = k[b, h // G, s], v[b, h // G, s], q[row, h * D:(h + 1) * D]
            logit = K @ x / math.sqrt(D)
            w = np.exp(logit - logit.max())
            w /= w.sum()
            o, a = w @ V, w @ np.abs(V)
            off = np.abs(got[row, h * D:(h + 1) * D] - o)
            tol = tol_of(o, a, c, np.abs(V).max(), (np.abs(K) @ np.abs(x)).max() / math.sqrt(D))
            assert np.isfinite(off).all(), f"row {row}, head {h}: not finite"
            assert (off <= tol).all(), f"row {row}, head {h}: off by {off.max()}, {np.max(off / tol)} of the tolerance"


def usual(D):
    """The tolerance of any keys: the weights' rounding besides, and scores summed in fp32."""
    return lambda o, a, c, v, size: equal_weights(o, a, c, v, size) + c * 2.0 ** -36 * v + 2 * (D + 2) * 2.0 ** -24 * size * a


def equal_weights(o, a, c, v, size):
    """Of keys whose scores are equal or too far apart to count: the weights' rounding to fp16, the sums' at most 64 roundings of 2^-24 and the
    result's to fp16, 2^-11 (2^-25 where it is subnormal)."""
    return 2.0 ** -11 * np.abs(o) + 2.0 ** -25 + (2.0 ** -11 + 64 * 2.0 ** -24) * a


@gpu
@pytest.mark.parametrize("exponent", [9, 11, 12, 15])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("members,shared,own", [(9, 700, 90), (2, 300, 500)])
def test_scores_past_fp32s_whole_numbers(torch_mod, dev, members, shared, own, D, exponent):
    """q is 2^exponent and K +-1.75 of it throughout, so every product and every sum of a score is exact in fp32 and its rounding after the scale
    is the same for all keys of one score: the keys of the greater score count alike, the others not at all."""
    case = Case([(members, shared), (1, 0)], [own, max(1, own // 3)], 8, 2, D, seed=members + D)
    r = np.random.default_rng(exponent)
    case.q[:] = f16_bits(np.float32(2.0 ** exponent))
    sign = np.where(r.random(case.k.shape[:3]) < 0.5, 1, -1).astype(np.float32)
    case.k[:] = f16_bits(np.broadcast_to(sign[..., None] * np.float32(1.75 * 2.0 ** exponent), case.k.shape))
    run(torch_mod, dev, case, equal_weights)


@gpu
@pytest.mark.parametrize("members", [9, 2])
@pytest.mark.parametrize("up", [True, False])
def test_scores_that_grow_or_fall_along_the_keys(torch_mod, dev, members, up):
    """Key j has K = 1.25 * 2^e with e from -14 to 15, up or down, 20 keys of each: scores from 2^4 to 2^33, doubled from one to the next, so that only
    the keys of the greatest count."""
    case = Case([(members, 520)], [80], 8, 2, 64, seed=members)
    case.q[:] = f16_bits(np.float32(2.0 ** 15))
    for rows in case.keys:
        for j, (b, s) in enumerate(rows):
            case.k[b, :, s] = f16_bits(np.float32(1.25 * 2.0 ** (j // 20 - 14 if up else 15 - j // 20)))
    run(torch_mod, dev, case, equal_weights)


@gpu
@pytest.mark.parametrize("members", [9, 2])
def test_scores_far_apart_in_one_wave(torch_mod, dev, members):
    """Heads of scores past 2^24, of either sign, beside heads of scores of up to 36. K is +-1.5 * 2^10 for kv head 0, 1.75 * 2^14 for kv head 1: exact sums
    and two scores, or one, for every row. Small scores have a score's usual error besides, and their smaller weights 2^-25."""
    case = Case([(members, 640)], [70], 8, 2, 64, seed=members)
    q, k, r = bits_to_f32(case.q).reshape(-1, 8, 64), bits_to_f32(case.k), np.random.default_rng(3)
    q[:, :3] = np.array([1, 2, 3])[:, None] * 2.0 ** -10
    q[:, 3] = 2.0 ** 15
    q[:, 5] = -2.0 ** 15
    k[:, 0] = np.where(r.random(k[:, 0].shape[:2]) < 0.3, 1, -1)[..., None] * 1.5 * 2.0 ** 10
    k[:, 1] = 1.75 * 2.0 ** 14
    case.q, case.k = f16_bits(q).reshape(case.q.shape), f16_bits(k)
    run(torch_mod, dev, case, lambda o, a, c, v, size: equal_weights(o, a, c, v, size) + (c * 2.0 ** -25 * v + 2 * 66 * 2.0 ** -24 * size * a if size < 100 else 0))


@gpu
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("members,shared,own,hints", [(9, 20000, 40, (9, 128, 40)), (2, 1000, 12000, (2, 128, 0)), (1, 0, 9000, (1, 0, 0)), (40, 6000, 20, None)])
def test_many_keys_far_below_one(torch_mod, dev, members, shared, own, hints, D):
    """Key 0 has a score of 18, value 0; all others 0, with values of one sign: e^-18 = 2^-26 of key 0's weight each, and all of the result.
    Each weight is rounded to fp16, 2^-11 of it, or 2^-25 of 2^-11 of the greatest where that is subnormal; scores are exact but for their
    scale (2 (D + 2) 2^-24 of their size); sums and result as elsewhere."""
    case = Case([(members, shared)], [own], 8, 2, D, seed=D + members)
    q, k, v = np.zeros((members, 8, D)), np.zeros(case.k.shape), np.abs(bits_to_f32(case.v)) + 0.25
    q[:, :, 0] = 2.0 * math.sqrt(D) if D != 128 else 22.625  # a score of 17.998 there
    for b, s in {rows[0] for rows in case.keys}:
        k[b, :, s, 0] = 9.0
        v[b, :, s] = 0.0
    case.q, case.k, case.v = f16_bits(q).reshape(case.q.shape), f16_bits(k), f16_bits(v)
    run(torch_mod, dev, case, lambda o, a, c, v, size: 2.0 ** -11 * np.abs(o) + 2.0 ** -25 + c * 2.0 ** -36 * v
        + (2.0 ** -11 + 2 * (D + 2) * 2.0 ** -24 * size + 64 * 2.0 ** -24) * a, hints=hints)


# (tokens, shared, own, heads, kv heads, head size), and us of rh_paged_decode_attention / this as measured
MEASURED = [
    ((16, 1024, 300, 16, 1, 128), 13.1, 14.2), ((64, 512, 100, 16, 1, 128), 13.6, 15.3), ((16, 2048, 40, 32, 2, 128), 16.0, 17.3),
    ((64, 512, 100, 32, 2, 128), 14.3, 17.1), ((64, 16, 60, 64, 4, 128), 6.9, 15.9), ((64, 512, 100, 12, 1, 128), 12.4, 14.7),
    ((48, 16, 4000, 32, 8, 128), 97.9, 107.8), ((48, 16, 4000, 32, 4, 64), 28.3, 32.6), ((2, 4096, 16000, 8, 8, 128), 23.6, 30.2),
    ((30, 2672, 267, 32, 1, 128), 24.9, 20.0), ((100, 7104, 142, 12, 1, 128), 52.8, 28.6), ((3, 3392, 3392, 64, 4, 128), 39.8, 19.6),
    ((87, 4864, 4864, 32, 1, 128), 125.1, 70.9), ((18, 16032, 320, 64, 4, 128), 72.3, 42.5), ((79, 17728, 1772, 32, 1, 128), 163.2, 61.8),
    ((5, 10176, 203, 64, 2, 128), 42.7, 23.2), ((104, 784, 1176, 28, 4, 128), 72.7, 42.1), ((14, 3776, 75, 8, 8, 64), 16.6, 12.7),
    ((51, 304, 152, 8, 8, 128), 19.1, 15.5), ((75, 5888, 5888, 16, 8, 32), 86.2, 67.5), ((120, 1008, 100, 28, 4, 128), 52.6, 22.7),
    ((48, 4096, 4000, 28, 4, 128), 102.0, 70.9), ((55, 352, 176, 8, 8, 128), 21.1, 16.3), ((4, 512, 100, 64, 2, 64), 9.6, 11.3),
    ((16, 512, 100, 40, 1, 32), 5.8, 10.0), ((16, 1024, 300, 40, 1, 32), 8.8, 10.3), ((16, 1024, 300, 12, 1, 128), 11.9, 14.1),
    ((16, 512, 100, 64, 2, 64), 8.0, 11.7), ((64, 16, 60, 40, 1, 64), 5.7, 10.7), ((16, 16, 60, 40, 1, 64), 5.5, 9.5),
    ((3, 13232, 19848, 8, 8, 64), 25.9, 30.1), ((27, 336, 33, 64, 8, 128), 13.6, 16.3), ((32, 1728, 864, 16, 4, 32), 10.4, 12.6),
    ((48, 4096, 16000, 9, 3, 64), 89.5, 104.6), ((8, 4176, 2088, 32, 4, 64), 12.2, 16.6), ((48, 16, 4000, 32, 4, 64), 28.1, 32.6),
    ((48, 16, 4000, 14, 2, 64), 19.3, 22.4)]


@pytest.mark.parametrize("shape,decode,shared", MEASURED)
def test_sharing_pays_says_what_was_measured(shape, decode, shared):
    assert _lib.lib().rh_shared_prefix_pays(*shape) == (shared < decode)


@pytest.mark.parametrize("shared", [1, 16, 16384, 1 << 30])
def test_one_token_shares_nothing(shared):
    for heads, kv_heads, D in ((16, 1, 128), (32, 8, 128), (40, 1, 64)):
        assert _lib.lib().rh_shared_prefix_pays(1, shared, 0, heads, kv_heads, D) == 0


@gpu
@pytest.mark.parametrize("D", [16, 64, 128])
def test_no_groups_at_all(torch_mod, dev, D):
    """Tokens on their own, with no group array: what rh_shared_prefix_groups leaves where nothing is shared."""
    case = Case([(1, 0)] * 7, [300, 1, 65, 1100], 8, 2, D, seed=D)
    want, tol = case.oracle()
    case.groups = []
    call = Call(torch_mod, dev, case)
    args = list(call.args)
    assert args[8] == 0
    args[5] = None
    _lib.check(call.lib.rh_shared_prefix_attention(*args, None))
    torch_mod.cuda.synchronize()
    assert (np.abs(call.out.double().cpu().numpy() - want) <= tol).all()


@gpu
@pytest.mark.parametrize("hints", [(2 ** 31 - 1, 2000, 300), (65536, 1 << 30, 1 << 30)])
@pytest.mark.parametrize("heads,kv_heads,D", [(32, 8, 128), (9, 3, 64)])
def test_hints_far_above_many_groups(torch_mod, dev, heads, kv_heads, D, hints):
    """A group has no more members than there are tokens: the largest numbers that the call takes for its sizes fit its launch."""
    run(torch_mod, dev, Case([(3, 160 + 16 * (i % 5)) for i in range(40)], [9, 40], heads, kv_heads, D, seed=D), usual(D), hints=hints)
