"""gsdlq_logprobs_rows against the definition in 64 bits."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def reference(x, temp):
    """z, log p and entropy in 64 bits.  The cleaned logit and its quotient are the operator's inputs' own values."""
    z = np.where(np.isnan(x), -1e4, np.where(np.isposinf(x), 100.0, np.where(np.isneginf(x), -1e4, x))).astype(np.float64)
    z = z / max(np.float32(temp), np.float32(1e-4)).astype(np.float64)
    m = z.max(1, keepdims=True)
    e = np.exp(z - m)
    lp = z - m - np.log(e.sum(1, keepdims=True))
    return z, lp, -(np.where(e > 0, np.exp(lp), 0.0) * lp).sum(1)


def run(x, ids=None, top=0, temp=1.0, entropy=True):
    from gsdlq_b200 import ops
    rows = x.shape[0]
    out = {}
    if ids is not None:
        out["ids"] = torch.tensor(ids, dtype=torch.int32, device="cuda")
        out["logprob"] = torch.full((rows,), 9.0, device="cuda")
    if entropy:
        out["entropy"] = torch.full((rows,), 9.0, device="cuda")
    if top:
        out["top_ids"] = torch.full((rows, top), -7, dtype=torch.int32, device="cuda")
        out["top_logprobs"] = torch.full((rows, top), 9.0, device="cuda")
    ops.logprobs_rows(ops.logprobs_job(x, temperature=temp, **out))
    return {k: v.cpu().numpy() for k, v in out.items()}


def check(x, ids, top, temp=1.0):
    import gsdlq_b200._lib as L
    xs = x.cpu().numpy()
    z, lp, ent = reference(xs, temp)
    got = run(x, ids, top, temp)
    n, size = xs.shape[1], np.abs(z).max(1)
    # z is off by half a step of its own, a difference z - m by the two and its own; each sum of n terms (a
    # thread's n / 128 of them at most, then a tree of 32 steps) by that many half steps; exp, log and their
    # argument by a few; the entropy's terms e^u u are at most 1/e each and so bounded by the same sums' errors.
    half = 2.0 ** -24
    tol = half * (6 * size + np.abs(lp).max(1) * 2 + n / 128 + 64) + 1e-45
    rows = np.arange(len(ids))
    known = np.array(ids) >= 0
    want = np.where(known, lp[rows, np.maximum(ids, 0)], 0.0)
    assert (np.abs(got["logprob"] - want) <= np.where(known, tol, 0.0)).all()
    assert (np.abs(got["entropy"] - ent) <= tol * (2 + np.abs(ent))).all()
    if top:
        zf = np.where(np.isnan(xs), np.float32(-1e4), np.where(np.isposinf(xs), np.float32(100), np.where(
            np.isneginf(xs), np.float32(-1e4), xs))) / max(np.float32(temp), np.float32(1e-4))
        order = np.argsort(-zf.astype(np.float32), axis=1, kind="stable")[:, :top]
        assert np.array_equal(got["top_ids"], order)
        assert (np.abs(got["top_logprobs"] - np.take_along_axis(lp, order, 1)) <= tol[:, None]).all()
    assert L.device_flags() == 0
    return got


@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (1, 2, 2), (3, 31, 31), (2, 32, 32), (5, 257, 5), (1, 32768, 20),
                                        (7, 1000, 32), (128, 4097, 8), (200, 515, 3), (2, 151936, 32), (16, 49152, 0),
                                        (1, 50257, 1), (300, 100, 20)])
def test_rows_sizes_and_alternatives(cuda_lib, rng, rows, n, top):
    x = torch.from_numpy(rng.standard_normal((rows, n)) * 3).float().cuda()
    ids = [int(i) for i in rng.integers(-1, n, rows)]
    for temp in (1.0, 0.6):
        check(x, ids, top, temp)


def test_equal_logits_and_many_ties(cuda_lib, rng):
    """Rows with no order among the tokens, and few distinct values: the lowest indices, in order."""
    for n in (40, 3001, 65537):
        x = torch.zeros((3, n), device="cuda")
        x[1] = -0.0
        x[1, ::2] = 0.0  # -0 and 0 are equal
        x[2] = torch.from_numpy(rng.integers(0, 3, n).astype(np.float32)).cuda()
        got = check(x, [0, n - 1, 5], 32)
        assert np.array_equal(got["top_ids"][0], np.arange(32)) and np.array_equal(got["top_ids"][1], np.arange(32))


def test_alternatives_crowded_in_one_place(cuda_lib, rng):
    """Thousands of tokens above all others, in rows that a block or a cluster reads so that a few threads hold them
    all; and rows with fewer unmasked tokens than alternatives."""
    for rows, n, part in ((1, 400000, 50000), (300, 151936, 151936)):
        x = torch.from_numpy(rng.standard_normal((rows, n)).astype(np.float32)).cuda()
        i = torch.arange(n, device="cuda") % part
        x += 100.0 * ((i // 4) % 512 < 24)
        got = check(x, [7] * rows, 5)
        assert ((got["top_ids"] % part // 4) % 512 < 24).all()
    x = torch.full((3, 151936), -math.inf, device="cuda")
    x[:, 77::50000] = torch.arange(12, device="cuda").float().reshape(3, 4)
    got = check(x, [77, 78, 150077], 30)
    assert np.array_equal(got["top_ids"][:, 4:], np.tile(np.r_[0:26], (3, 1)))


def test_masked_and_non_finite_logits(cuda_lib, rng):
    """Masked tokens (-inf, the type's lowest value), NaN and +inf follow the sampler's rules; a row in which
    everything is masked is uniform."""
    x = torch.from_numpy(rng.standard_normal((8, 700)) * 2).float().cuda()
    low = torch.finfo(torch.float32).min
    x[0, 100:] = -math.inf
    x[1, 1:] = low
    x[2] = -math.inf
    x[3] = math.nan
    x[4, 7] = math.inf
    x[5, ::3] = math.nan
    x[6] = low
    x[7, :650] = low
    got = check(x, [3, 0, 699, 5, 7, 1, 2, 699], 10)
    assert np.allclose(got["entropy"][[2, 3, 6]], math.log(700), rtol=1e-6)
    # a quotient past the type's range: finite results or -inf, never NaN
    for temp in (1e-4, 1e-30):
        got = run(x, [3, 0, 0, 5, 7, 1, 2, 699], 10, temp)
        assert not any(np.isnan(v).any() for v in got.values())


@pytest.mark.parametrize("rows,n", [(3, 700), (2, 151936), (200, 4097)])
def test_alternatives_among_quotients_past_the_range(cuda_lib, rng, rows, n):
    """Rows with fewer unmasked tokens than alternatives, masked with the type's lowest value or another value whose
    quotient is past the type's range, count those quotients as -FLT_MAX: equal, in order of their indices."""
    big = np.float32(np.finfo(np.float32).max)
    for temp in (0.5, 0.9999, 1e-4, 1.0, 2.0):
        x = torch.full((rows, n), -float(big), device="cuda")
        x[:, 5::7] = -float(big) * 0.75
        for r in range(rows):
            x[r, torch.from_numpy(rng.permutation(n)[:r % 4])] = torch.from_numpy(
                rng.standard_normal(r % 4).astype(np.float32)).cuda()
        got = run(x, list(range(rows)), 20, temp)
        xs = x.cpu().numpy()
        with np.errstate(over="ignore"):
            z = np.clip(xs / np.float32(temp), -big, big)
        order = np.argsort(-z, axis=1, kind="stable")[:, :20]
        assert np.array_equal(got["top_ids"], order), temp
        for r in range(rows):
            assert np.isfinite(got["top_logprobs"][r, :r % 4]).all()
            assert (got["top_logprobs"][r, 1:] <= got["top_logprobs"][r, :-1]).all()


def test_alternatives_whose_quotients_are_subnormal(cuda_lib, rng):
    """At temperatures that leave a quotient few bits, many different logits share one and go by their indices."""
    for rows, n in ((4, 900), (2, 70001)):
        x = torch.from_numpy(rng.standard_normal((rows, n)) * 2).float().cuda()
        for temp in (1e30, 1e37, 3e38):
            xs = (x * 1e-7 if temp > 1e36 else x).cpu().numpy()
            z = xs / np.float32(temp)
            got = run(torch.from_numpy(xs).cuda(), None, 32, temp)
            assert np.array_equal(got["top_ids"], np.argsort(-z, axis=1, kind="stable")[:, :32]), temp


def test_peaked_rows_keep_their_small_numbers(cuda_lib):
    """Where nearly all probability is on one token, its log probability and the entropy are far below 1 and keep
    their leading digits: relative error of the sums 2^-24 (n / 128 + 64), of e^u 2^-23 (|u| + 2)."""
    x = torch.full((1, 512), -30.0, device="cuda")
    x[0, 77] = 0.0
    got = run(x, [77], 1)
    s = 511 * math.exp(-30.0)
    rel = 2.0 ** -24 * (512 / 128 + 64) + 2.0 ** -23 * 32
    assert abs(got["logprob"][0] + math.log1p(s)) <= rel * s
    ent = math.log1p(s) + 30.0 * s / (1 + s)
    assert abs(got["entropy"][0] - ent) <= 2 * rel * ent
    assert got["top_ids"][0, 0] == 77


def test_strided_rows_and_parts_of_the_output(cuda_lib, rng):
    wide = torch.from_numpy(rng.standard_normal((5, 1003))).float().cuda()
    for lo, n in ((0, 1000), (1, 999), (2, 500), (3, 1000)):  # rows that start at any 4-byte boundary
        check(wide[:, lo:lo + n], [0, -1, n - 1, 1, 2], 7)
    x = wide[:, :1000]
    full = run(x, [1, 2, 3, 4, 5], 6)
    for kw in (dict(ids=[1, 2, 3, 4, 5], entropy=False), dict(entropy=True), dict(top=6, entropy=False)):
        part = run(x, **kw)
        for k, v in part.items():
            assert np.array_equal(v, full[k]), k


def test_bad_token_ids_are_reported(cuda_lib, rng):
    import gsdlq_b200._lib as L
    x = torch.from_numpy(rng.standard_normal((4, 50))).float().cuda()
    got = run(x, [50, -2, 2**31 - 1, 49])
    assert got["logprob"][:3].tolist() == [0, 0, 0] and got["logprob"][3] < 0
    assert L.flag_names(L.device_flags()) == ["bad_token"]


def test_same_result_in_a_graph_and_run_to_run(cuda_lib, rng):
    from gsdlq_b200 import ops
    x = torch.from_numpy(rng.standard_normal((3, 20000)) * 4).float().cuda()
    ent, ids, lps = (torch.zeros(3, device="cuda"), torch.zeros((3, 9), dtype=torch.int32, device="cuda"),
                     torch.zeros((3, 9), device="cuda"))
    job = ops.logprobs_job(x, entropy=ent, top_ids=ids, top_logprobs=lps)
    ops.logprobs_rows(job)
    first = [t.clone() for t in (ent, ids, lps)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.logprobs_rows(job)
    for t in (ent, ids, lps):
        t.zero_()
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(first, (ent, ids, lps)))
