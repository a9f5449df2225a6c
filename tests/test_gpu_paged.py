"""The paged cache's operators on the GPU (gsdlq_rope_kv_paged, gsdlq_attention_paged, gsdlq_pages_*) against
plain restatements (paged_oracle.py): page bookkeeping and stored rows exactly, attention within a bound derived
there.  Everything of a pool that no position uses is NaN, so that a read of it shows."""
import math

import numpy as np
import pytest

import paged_oracle as O

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def flags():
    import gsdlq_b200._lib as L
    return L.flag_names(L.device_flags())


def dev(a, dtype=torch.int32):
    return torch.tensor(a, dtype=dtype, device="cuda")


def make_pool(rng, lens, page, nkv, hd, dtype, layers=1, spare=3, max_blocks=None):
    """Sequences of the given lengths over shuffled pages; all else NaN."""
    from gsdlq_b200 import paged
    blocks = [-(-n // page) for n in lens]
    n_pages, mb = sum(blocks) + spare, max_blocks or max(blocks) + 1
    perm = rng.permutation(n_pages)
    table = np.full((len(lens), mb), -1, np.int64)
    refs = np.zeros(n_pages, np.int64)
    k = torch.full((layers, n_pages, page, nkv, hd), math.nan, dtype=dtype)
    v = k.clone()
    at = 0
    for s, (n, b) in enumerate(zip(lens, blocks)):
        table[s, :b] = perm[at:at + b]
        refs[perm[at:at + b]] = 1
        for j in range(b):
            m = min(page, n - j * page)
            for t in (k, v):
                t[:, perm[at + j], :m] = torch.from_numpy(rng.standard_normal((layers, m, nkv, hd))).to(dtype)
        at += b
    return paged.PagedKV.wrap(k.cuda(), v.cuda(), dev(table), dev(refs))


def rows_of(kv, layer, seq, n):
    """K and V of a sequence's first n positions, as float64."""
    out = []
    for t in (kv.k, kv.v):
        pages = kv.table[seq, :-(-n // kv.page_size)].long()
        out.append(t[layer, pages].flatten(0, 1)[:n].double().cpu().numpy())
    return out


def run_attention(kv, layer, q, pos, row_seq=None, scale=None):
    from gsdlq_b200 import ops
    rows, heads, hd = q.shape
    guard = torch.full((rows + 1, heads, hd), 77.0, device="cuda")
    job = ops.paged_attn_job(kv, layer, q, guard[:rows], dev(pos), scale or 1.0 / math.sqrt(hd),
                             ops.attention_paged_work(kv, rows, heads), None if row_seq is None else dev(row_seq))
    ops.attention_paged(job)
    first = guard[:rows].clone()
    ops.attention_paged(job)  # the work area serves the next launch, with the same result
    assert torch.equal(first, guard[:rows]) and bool((guard[rows] == 77.0).all())
    return first.cpu().numpy()


def check_attention(kv, layer, q, pos, row_seq=None, scale=None):
    got = run_attention(kv, layer, q, pos, row_seq, scale)
    for r, p in enumerate(pos):
        k, v = rows_of(kv, layer, r if row_seq is None else row_seq[r], p + 1)
        want, tol = O.attention(q[r].cpu().numpy(), k, v, scale or 1.0 / math.sqrt(q.shape[2]))
        err = np.abs(got[r] - want)
        assert (err <= tol).all(), (r, p, float((err - tol).max()), float(err.max()))
        if p < 0:
            assert not got[r].any()
    assert flags() == []


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hd,nkv,group,page", [
    (128, 2, 4, 16), (128, 1, 1, 64), (64, 4, 1, 16), (64, 2, 3, 5), (32, 3, 8, 1), (128, 2, 6, 100), (64, 1, 12, 24),
    (32, 7, 1, 32), (128, 1, 17, 48)])
def test_attention_lengths_groups_and_pages(cuda_lib, rng, kind, hd, nkv, group, page):
    lens = [1, 2, 15, 16, 17, 0, 31, 33, 63, 64, 65, 0, 127, 130, 257, 600]
    kv = make_pool(rng, lens, page, nkv, hd, DTYPES[kind], layers=2)
    q = torch.from_numpy(rng.standard_normal((len(lens), nkv * group, hd)) * 2).float().cuda()
    check_attention(kv, 1, q, [n - 1 for n in lens])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attention_single_rows_over_long_caches(cuda_lib, rng, kind):
    for hd, nkv, group, n in ((128, 1, 4, 9001), (64, 3, 2, 4097), (32, 1, 5, 7000), (128, 8, 4, 1537)):
        kv = make_pool(rng, [n], 16, nkv, hd, DTYPES[kind])
        q = torch.from_numpy(rng.standard_normal((1, nkv * group, hd)) * 2).float().cuda()
        for pos in (n - 1, n // 2, 0):
            check_attention(kv, 0, q, [pos])


def test_attention_chunk_rows_and_repeated_sequences(cuda_lib, rng):
    """Consecutive positions of one sequence, rows of several sequences in any order, and the same row twice."""
    kv = make_pool(rng, [300, 40], 16, 2, 128, torch.float16)
    rows = [(0, 290 + i) for i in range(10)] + [(1, 3), (0, 7), (1, 39), (1, -1), (0, 7)]
    q = torch.from_numpy(rng.standard_normal((len(rows), 12, 128)) * 2).float().cuda()
    q[14] = q[11]
    pos, seq = [p for _, p in rows], [s for s, _ in rows]
    check_attention(kv, 0, q, pos, seq)
    got = run_attention(kv, 0, q, pos, seq)
    assert np.array_equal(got[11], got[14])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hd,nkv,group,page", [(128, 2, 6, 16), (64, 4, 1, 24), (32, 2, 2, 1), (64, 2, 3, 16),
                                               (128, 1, 4, 64), (64, 1, 8, 7), (32, 1, 20, 16)])
def test_attention_many_rows_of_few_sequences(cuda_lib, rng, kind, hd, nkv, group, page):
    """Packs of rows: whole chunks of sequences, idle rows and changes of sequence inside them, positions in any
    order, more rows than a block counts at once."""
    kv = make_pool(rng, [211, 70, 1], page, nkv, hd, DTYPES[kind], layers=2)
    rows = [(0, p) for p in range(150, 211)] + [(1, 69 - p) for p in range(33)] + [(2, 0)] * 3 + [(1, -1)] * 2
    rows += [(int(rng.integers(0, 3)), int(rng.integers(-1, 1))) for _ in range(20)]
    rows += [(0, int(p)) for p in rng.integers(-1, 211, 50)]
    q = torch.from_numpy(rng.standard_normal((len(rows), nkv * group, hd)) * 2).float().cuda()
    check_attention(kv, 1, q, [p for _, p in rows], [s for s, _ in rows])


def test_attention_hundreds_of_sequences(cuda_lib, rng):
    """More rows than a block counts at once, each of a sequence of its own, in order and permuted."""
    n = 300
    lens = [int(x) for x in rng.integers(0, 90, n)]
    lens[7], lens[200] = 700, 1300
    kv = make_pool(rng, lens, 16, 2, 64, torch.float16)
    q = torch.from_numpy(rng.standard_normal((n, 6, 64)) * 2).float().cuda()
    check_attention(kv, 0, q, [x - 1 for x in lens])
    seq = [int(s) for s in rng.permutation(n)]
    check_attention(kv, 0, q, [lens[s] - 1 for s in seq], seq)
    check_attention(kv, 0, q[:40], [lens[s] - 1 for s in seq[:40]], seq[:40])


def test_attention_chunks_over_long_caches(cuda_lib, rng):
    """Chunks split over many blocks and joined; the last rows of a chunk see what the first ones do not."""
    for hd, nkv, group, n in ((128, 2, 6, 3001), (64, 3, 1, 5000), (32, 1, 4, 4100)):
        kv = make_pool(rng, [n], 16, nkv, hd, torch.float16)
        for rows in (2, 5, 37, 128):
            pos = list(range(n - rows, n))
            q = torch.from_numpy(rng.standard_normal((rows, nkv * group, hd)) * 2).float().cuda()
            check_attention(kv, 0, q, pos, [0] * rows)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hd,nkv,group,page", [(128, 2, 6, 16), (64, 32, 1, 16), (32, 8, 2, 5), (128, 8, 4, 48)])
def test_a_row_never_meets_what_lies_behind_it(cuda_lib, rng, kind, hd, nkv, group, page):
    """Cache rows that are not finite, in use by later rows of the call: the rows before them, in the same pack of rows
    and elsewhere, are as they are without; idle rows among them are zero."""
    n = 2100
    kv = make_pool(rng, [n], page, nkv, hd, DTYPES[kind])
    k, v = rows_of(kv, 0, 0, n)
    wild = {1300: math.inf, 2040: -math.inf, 2041: math.nan, 2063: math.inf, 2095: math.nan}
    for t, x in wild.items():
        at = (0, int(kv.table[0, t // page]), t % page, int(rng.integers(0, nkv)), int(rng.integers(0, hd)))
        kv.v[at] = x
        if t % 2:
            kv.k[at] = x
    from gsdlq_b200 import ops

    def run(q, pos):  # (run_attention's comparison of two launches has no use for NaN)
        out = torch.full_like(q, 77.0)
        ops.attention_paged(ops.paged_attn_job(kv, 0, q, out, dev(pos), hd ** -0.5,
                                               ops.attention_paged_work(kv, len(pos), q.shape[1]), dev([0] * len(pos))))
        return out.cpu().numpy()

    cases = [list(range(n - 128, n)),                                     # the last chunk of a prompt
             list(range(1290, 1311)) * 7,                                 # short packs, over again
             [2039 - r if r % 3 else 2099 - r for r in range(130)],       # ends far apart and in any order
             [int(p) for p in rng.integers(-1, n, 200)]]                  # idle rows too
    for pos in cases:
        q = torch.from_numpy(rng.standard_normal((len(pos), nkv * group, hd)) * 2).float().cuda()
        for rows in (slice(None), slice(0, 2)):  # tiles shared by many rows, and a tile per row
            got = run(q[rows], pos[rows])
            clean = [r for r, p in enumerate(pos[rows]) if p < 1300]
            assert np.isfinite(got[clean]).all()
            for r in clean[::8]:
                p = pos[r]
                want, tol = O.attention(q[r].cpu().numpy(), k[:p + 1], v[:p + 1], hd ** -0.5)
                assert (np.abs(got[r] - want) <= tol).all(), (r, p)
    # the first of them gone: the rows up to the second
    at = (0, int(kv.table[0, 1300 // page]), 1300 % page)
    kv.v[at] = torch.from_numpy(v[1300]).to(kv.v.dtype).cuda()
    for pos in cases[0], cases[2], cases[3]:
        q = torch.from_numpy(rng.standard_normal((len(pos), nkv * group, hd)) * 2).float().cuda()
        got = run(q, pos)
        for r, p in enumerate(pos):
            if p < 2040:
                assert np.isfinite(got[r]).all(), (r, p)
                if r % 8 == 0 or p > 2030:
                    want, tol = O.attention(q[r].cpu().numpy(), k[:p + 1], v[:p + 1], hd ** -0.5)
                    assert (np.abs(got[r] - want) <= tol).all(), (r, p)
            elif p >= 2041:  # position 2041's NaN in K and V is its own
                assert np.isnan(got[r]).any(), (r, p)
    assert flags() == []


def test_one_work_area_serves_launches_of_any_shape_in_turn(cuda_lib, rng):
    """Launches of few and many rows, in both forms and of all head sizes, on one work area: each the same bit for bit
    as with a work area of its own, with every row written, and within the bound."""
    from gsdlq_b200 import ops, paged
    shared = None
    for hd, nkv, group in ((64, 32, 1), (128, 8, 4), (32, 8, 1), (64, 32, 1)):
        one = make_pool(rng, [1260], 16, nkv, hd, torch.float16)
        table = torch.full((400, one.max_blocks), -1, dtype=torch.int32, device="cuda")
        table[0] = one.table[0]
        many = paged.PagedKV.wrap(one.k, one.v, table, one.refs)  # as many sequences: a tile per row
        heads = nkv * group
        if shared is None:
            shared = ops.attention_paged_work(one, 300, 32)
        for rows in (30, 128, 6, 128, 2, 64, 300, 1, 128):
            q = torch.from_numpy(rng.standard_normal((rows, heads, hd)) * 2).float().cuda()
            pos, seq = [900 + r for r in range(rows)], dev([0] * rows)
            for kv in (one, many):
                outs = []
                for work in (shared, ops.attention_paged_work(kv, rows, heads)):
                    out = torch.full((rows, heads, hd), math.nan, device="cuda")
                    ops.attention_paged(ops.paged_attn_job(kv, 0, q, out, dev(pos), hd ** -0.5, work, seq))
                    outs.append(out.cpu().numpy())
                assert np.array_equal(outs[0], outs[1]), (hd, rows, kv is one)
                for r in {0, rows // 2, rows - 1}:
                    k, v = rows_of(kv, 0, 0, pos[r] + 1)
                    want, tol = O.attention(q[r].cpu().numpy(), k, v, hd ** -0.5)
                    assert (np.abs(outs[0][r] - want) <= tol).all(), (hd, rows, r)
    assert flags() == []


def test_a_chunk_of_one_sequence_through_a_table_of_its_own(cuda_lib, rng):
    """As the documents say for one sequence out of many: append and attention over a cache of that sequence alone, which
    shares pool, table and counts with the others'."""
    from gsdlq_b200 import paged
    kv = make_pool(rng, [90, 200, 17, 40], 16, 4, 64, torch.float16)
    alone = paged.PagedKV.wrap(kv.k, kv.v, kv.table[1:2], kv.refs)
    pos = list(range(100, 200))
    append_check(alone, 0, rng, pos, 8, row_seq=[0] * 100)
    q = torch.from_numpy(rng.standard_normal((100, 8, 64))).float().cuda()
    check_attention(alone, 0, q, pos, [0] * 100)
    check_attention(kv, 0, q[-1:].repeat(4, 1, 1), [89, 199, 16, 39])


def test_attention_strided_q_and_extreme_scores(cuda_lib, rng):
    kv = make_pool(rng, [50, 200, 7], 16, 2, 64, torch.float16)
    wide = torch.from_numpy(rng.standard_normal((3, 4 * 64 + 20))).float().cuda()
    q = wide[:, :256].unflatten(1, (4, 64))
    check_attention(kv, 0, q, [49, 199, 6])
    # one position far ahead of the others, scores of some hundreds, tiny queries and zero queries
    q = q.contiguous()
    q[0] *= 200.0
    q[1] *= 1e-30
    q[2] = 0.0
    check_attention(kv, 0, q, [49, 199, 6])
    check_attention(kv, 0, q, [49, 199, 6], scale=-0.25)


def test_attention_leaves_out_missing_pages(cuda_lib, rng):
    """A table entry outside the pool: its positions are left out and reported; no position left: zeros."""
    kv = make_pool(rng, [64, 64, 16], 16, 1, 64, torch.float16)
    q = torch.from_numpy(rng.standard_normal((3, 2, 64))).float().cuda()
    k, v = rows_of(kv, 0, 0, 64)
    keep = np.r_[0:16, 32:64]
    kv.table[0, 1] = -1
    kv.table[1] = torch.tensor([kv.n_pages, -7, 1 << 30, -(1 << 31)] + [-1] * (kv.max_blocks - 4), dtype=torch.int32)
    got = run_attention(kv, 0, q, [63, 63, 15])
    want, tol = O.attention(q[0].cpu().numpy(), k[keep], v[keep], 0.125)
    assert (np.abs(got[0] - want) <= tol).all() and not got[1].any()
    k, v = rows_of(kv, 0, 2, 16)
    want, tol = O.attention(q[2].cpu().numpy(), k, v, 0.125)
    assert (np.abs(got[2] - want) <= tol).all()
    assert flags() == ["bad_page"]
    # positions and sequences out of range are idle rows, and reported
    assert not run_attention(kv, 0, q, [-2, kv.max_blocks * 16, 2**31 - 1]).any()
    assert flags() == ["bad_pos"]
    assert not run_attention(kv, 0, q, [3, 3, 3], [-1, 3, 2**31 - 1]).any()
    assert flags() == ["bad_page"]
    # the same in the form for rows that share sequences (here six and more of three)
    q = q.repeat(3, 1, 1)
    got = run_attention(kv, 0, q, [63, 63, 15, 62, 1, -2, kv.max_blocks * 16, 2, 2], [0, 1, 2, 0, 0, 0, 0, 3, -1])
    k, v = rows_of(kv, 0, 2, 16)
    want, tol = O.attention(q[2].cpu().numpy(), k, v, 0.125)
    assert (np.abs(got[2] - want) <= tol).all() and not got[1].any() and not got[5:].any()
    k, v = (t[0, kv.table[0, [0, 2, 3]].long()].flatten(0, 1).double().cpu().numpy() for t in (kv.k, kv.v))
    for r, n in ((0, 48), (3, 47), (4, 2)):
        want, tol = O.attention(q[r].cpu().numpy(), k[:n], v[:n], 0.125)
        assert (np.abs(got[r] - want) <= tol).all()
    assert set(flags()) == {"bad_page", "bad_pos"}


def test_attention_of_chunks_leaves_out_missing_pages(cuda_lib, rng):
    """The same where enough rows share sequences to share tiles."""
    kv = make_pool(rng, [64, 64, 16], 16, 4, 64, torch.float16)
    k, v = rows_of(kv, 0, 0, 64)
    k2, v2 = rows_of(kv, 0, 2, 16)
    keep = np.r_[0:16, 32:64]
    kv.table[0, 1] = -1
    kv.table[1] = torch.tensor([kv.n_pages, -7, 1 << 30, -(1 << 31)] + [-1] * (kv.max_blocks - 4), dtype=torch.int32)
    rows = [(0, 63), (0, 62), (1, 63), (1, 5), (2, 15), (2, 3), (0, -2), (0, kv.max_blocks * 16), (3, 2), (-1, 2)] * 4
    q = torch.from_numpy(rng.standard_normal((len(rows), 4, 64))).float().cuda()
    got = run_attention(kv, 0, q, [p for _, p in rows], [s for s, _ in rows])
    for r, (s, p) in enumerate(rows):
        if s in (1, 3, -1) or p not in range(64):
            assert not got[r].any()
            continue
        n = keep[keep <= p] if s == 0 else np.arange(p + 1)
        want, tol = O.attention(q[r].cpu().numpy(), (k if s == 0 else k2)[n], (v if s == 0 else v2)[n], 0.125)
        assert (np.abs(got[r] - want) <= tol).all(), r
    assert set(flags()) == {"bad_page", "bad_pos"}


def test_attention_offsets_past_32_bits(cuda_lib, rng):
    """Pages whose elements lie more than 2^32 behind the start of the pool."""
    from gsdlq_b200 import paged
    page, nkv, hd = 64, 8, 128
    n_pages = (1 << 32) // (page * nkv * hd) + 40
    k = torch.empty((1, n_pages, page, nkv, hd), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    kv = paged.PagedKV.wrap(k, v, dev([[n_pages - 1, 3, n_pages - 30]]), dev(np.zeros(n_pages, np.int64)))
    for p in (n_pages - 1, 3, n_pages - 30):
        for t in (k, v):
            t[0, p] = torch.from_numpy(rng.standard_normal((page, nkv, hd))).to(torch.bfloat16)
    q = torch.from_numpy(rng.standard_normal((1, 32, hd))).float().cuda()
    check_attention(kv, 0, q, [170])
    kv.refs[n_pages - 30] = 1
    append_check(kv, 0, rng, [190], 32)
    kv.counts[0] = 1
    kv.copy_pages(dev([n_pages - 1]), dev([5]), kv.counts)
    assert torch.equal(k[0, 5], k[0, n_pages - 1]) and flags() == []


# ---------------------------------------------------------------------------------------- append
def append_check(kv, layer, rng, pos, heads, row_seq=None, interleaved=True, strided=False, in_place=False,
                 stored=None, max_pos=None):
    """Append random rows; the whole pool and q must be what the restatement gives (rows in ``stored`` are stored,
    by default those that are not idle)."""
    from gsdlq_b200 import ops
    rows, nkv, hd = len(pos), kv.n_kv_heads, kv.head_dim
    width = (heads + 2 * nkv) * hd
    qkv = torch.from_numpy(rng.standard_normal((rows, width + (12 if strided else 0)))).float().cuda()
    parts = [t.unflatten(1, (-1, hd)) for t in qkv[:, :width].split((heads * hd, nkv * hd, nkv * hd), 1)]
    q, k, v = parts if strided else [t.contiguous() for t in parts]
    want_q, nk, nv = (t.cpu().numpy().copy() for t in (q, k, v))
    cs = rng.standard_normal((max_pos or kv.max_blocks * kv.page_size, hd // 2, 2)).astype(np.float32)
    before = [t.clone() for t in (kv.k, kv.v)]
    out = q if in_place else torch.full_like(q, 5.0)
    ops.rope_kv_paged(ops.paged_append_job(kv, layer, q, k, v, out, dev(pos), torch.from_numpy(cs).cuda(),
                                           None if row_seq is None else dev(row_seq), interleaved))
    for r, p in enumerate(pos):
        s = r if row_seq is None else row_seq[r]
        if not 0 <= p < cs.shape[0] or p >= kv.max_blocks * kv.page_size or not 0 <= s < kv.n_seqs:
            continue
        want_q[r] = O.rotate(want_q[r], cs[p], interleaved)
        if stored is not None and r not in stored:
            continue
        page, o = int(kv.table[s, p // kv.page_size]), p % kv.page_size
        before[0][layer, page, o] = torch.from_numpy(O.rotate(nk[r], cs[p], interleaved)).to(kv.k.dtype)
        before[1][layer, page, o] = torch.from_numpy(nv[r]).to(kv.k.dtype)
    assert np.array_equal(out.cpu().numpy(), want_q)
    for got, want in zip((kv.k, kv.v), before):
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hd,nkv,heads,page", [(128, 2, 8, 16), (64, 32, 32, 24), (32, 3, 9, 1), (64, 5, 15, 64)])
def test_append_rows(cuda_lib, rng, kind, hd, nkv, heads, page):
    lens = [1, 33, 16, 5, 17, 64]
    kv = make_pool(rng, lens, page, nkv, hd, DTYPES[kind], layers=2)
    pos = [n - 1 for n in lens]
    pos[3] = -1
    append_check(kv, 1, rng, pos, heads)
    append_check(kv, 0, rng, pos, heads, strided=True)
    append_check(kv, 0, rng, pos, heads, interleaved=False, in_place=True)
    append_check(kv, 1, rng, [60, 61, 62, 63, 2], heads, row_seq=[5, 5, 5, 5, 1], strided=True, in_place=True)
    assert flags() == []


def test_append_in_place_with_the_packed_stride_given_or_not(cuda_lib, rng):
    """0 and the packed stride are the same stride, also where q is rotated in place."""
    from gsdlq_b200 import ops
    kv = make_pool(rng, [20, 20, 20], 16, 2, 64, torch.float16)
    q0 = torch.from_numpy(rng.standard_normal((3, 4, 64))).float().cuda()
    k = torch.from_numpy(rng.standard_normal((3, 2, 64))).float().cuda()
    cs = torch.from_numpy(rng.standard_normal((32, 32, 2))).float().cuda()
    got = []
    for q_stride, out_stride in ((0, 0), (0, 256), (256, 0), (256, 256)):
        q = q0.clone()
        job = ops.paged_append_job(kv, 0, q, k, k, q, dev([19, 18, 3]), cs)
        job.q_stride, job.q_out_stride = q_stride, out_stride
        ops.rope_kv_paged(job)
        got.append(q)
    assert all(torch.equal(got[0], x) for x in got[1:]) and not torch.equal(got[0], q0)
    assert flags() == []


def test_append_refuses_shared_and_missing_pages(cuda_lib, rng):
    kv = make_pool(rng, [20, 20, 20, 20], 16, 2, 64, torch.float16)
    kv.refs[int(kv.table[0, 1])] = 2   # shared
    kv.table[1, 1] = -1                # missing
    kv.table[2, 1] = kv.n_pages        # outside the pool
    append_check(kv, 0, rng, [19] * 4, 4, stored=[3])
    assert flags() == ["bad_page"]
    append_check(kv, 0, rng, [-1, -5, kv.max_blocks * 16, 5], 4)
    assert flags() == ["bad_pos"]
    append_check(kv, 0, rng, [3, 12, 3, 11], 4, max_pos=12)  # the table of angles ends at 12
    assert flags() == ["bad_pos"]
    append_check(kv, 0, rng, [3, 3, 3], 4, row_seq=[4, -1, 3])
    assert flags() == ["bad_page"]


def test_append_rounds_overflow_and_ties_as_the_type_does(cuda_lib, rng):
    from gsdlq_b200 import ops
    for dtype in DTYPES.values():
        kv = make_pool(rng, [16], 16, 1, 32, dtype)
        v = torch.tensor([65504.0, 65519.9, 65520.0, -1e30, 1e-8, 2.0**-24, 2.0**-25, 1.0 + 2.0**-11,
                          1.0 + 3 * 2.0**-11, 1.0 + 2.0**-8, 1.0 + 3 * 2.0**-8, 3.4e38, math.inf, -math.inf, 0.0, -0.0]
                         * 2, device="cuda").reshape(1, 1, 32)
        q = torch.zeros(1, 1, 32, device="cuda")
        cs = torch.zeros(16, 16, 2, device="cuda")
        cs[..., 0] = 1.0
        ops.rope_kv_paged(ops.paged_append_job(kv, 0, q, q.clone(), v, q.clone(), dev([15]), cs))
        got = kv.v[0, int(kv.table[0, 0]), 15, 0]
        assert torch.equal(got.view(torch.int16), v[0, 0].to(dtype).view(torch.int16))


# ---------------------------------------------------------------------------------------- pages
def empty_pool(n_pages, page, seqs, blocks, layers=2, dtype=torch.float16):
    """Every page of every layer holds values of its own."""
    from gsdlq_b200 import paged
    kv = paged.PagedKV(layers, n_pages, page, 2, 32, seqs, blocks, dtype)
    for t, sign in ((kv.k, 1), (kv.v, -1)):
        p = torch.arange(layers * n_pages, device="cuda").reshape(layers, n_pages, 1, 1, 1)
        t += (sign * (p % 997) + torch.arange(2 * 32, device="cuda").reshape(1, 1, 1, 2, 32) / 64).to(dtype)
    return kv


def same(kv, want, pools):
    assert kv.table.tolist() == want.table
    assert kv.refs.tolist() == want.refs
    for got, exp in zip((kv.k, kv.v), pools):
        assert torch.equal(got, exp)


def test_pages_random_sequences_of_operations(cuda_lib, rng):
    """Forks, reservations and compactions in random order on a pool that now and then runs out."""
    seqs, blocks, page, n_pages = 9, 11, 4, 40
    kv = empty_pool(n_pages, page, seqs, blocks)
    want = O.Pages(kv.table.tolist(), kv.refs.tolist(), page)
    pools = [kv.k.clone(), kv.v.clone()]

    def moved(pairs, counts, most):
        assert kv.counts[:3].tolist() == counts
        assert kv.src[:most].tolist() == [a for a, _ in pairs] + [-1] * (most - len(pairs))
        assert kv.dst[:most].tolist() == [b for _, b in pairs] + [-1] * (most - len(pairs))
        for t in pools:
            t[:, [b for _, b in pairs]] = t[:, [a for a, _ in pairs]].clone()

    ran_out = 0
    for step in range(150):
        what = rng.integers(0, 10)
        if what < 6:
            n = int(rng.integers(1, 3 * seqs))
            rows = [(int(rng.integers(0, seqs)), int(rng.integers(-1, blocks * page))) for _ in range(n)]
            kv.reserve(dev([p for _, p in rows]), dev([s for s, _ in rows]))
            pairs, failed, taken = want.reserve(rows)
            moved(pairs, [len(pairs), failed, taken], n)
            ran_out += failed > 0
            assert flags() == (["no_page"] if failed else [])
        elif what < 9:
            parent = [int(rng.choice([b, b, b, -1, rng.integers(0, seqs)])) for b in range(seqs)]
            kv.fork(dev(parent))
            want.fork(parent)
        else:
            most = int(rng.integers(1, 12))
            kv.compact(most)
            pairs, live, high = want.compact(most)
            moved(pairs, [len(pairs), live, high], most)
        same(kv, want, pools)
    assert ran_out > 3 and flags() == []


@pytest.mark.parametrize("n_pages", [1, 31, 4095, 4096, 4097, 20000, 270001])
def test_pages_large_pools_and_many_rows(cuda_lib, rng, n_pages):
    """Pools over several scan steps; free pages far apart; a thousand rows."""
    from gsdlq_b200 import paged
    seqs, blocks = 1024, 8
    refs = (rng.random(n_pages) < 0.7).astype(np.int64)
    kv = paged.PagedKV(1, n_pages, 2, 1, 32, seqs, blocks)
    kv.k += torch.arange(n_pages, device="cuda").reshape(1, -1, 1, 1, 1) % 1999
    live = np.flatnonzero(refs)
    flat = np.full(seqs * blocks, -1)
    flat[:min(len(live), flat.size)] = rng.permutation(live)[:flat.size]
    table = rng.permutation(flat).reshape(seqs, blocks)
    kv.table.copy_(dev(table))
    kv.refs.copy_(dev(refs))
    want = O.Pages(table, refs, 2)
    pools = [kv.k.clone(), kv.v.clone()]
    pos = [int(p) for p in rng.integers(-1, blocks * 2, seqs)]
    kv.reserve(dev(pos))
    pairs, failed, taken = want.reserve(list(enumerate(pos)))
    assert kv.counts[:3].tolist() == [len(pairs), failed, taken]
    same(kv, want, pools)
    kv.fork(dev([b // 2 if b % 3 else -1 for b in range(seqs)]))
    want.fork([b // 2 if b % 3 else -1 for b in range(seqs)])
    same(kv, want, pools)
    kv.compact()
    # the restatement's compaction, done at once
    live = [p for p, r in enumerate(want.refs) if r > 0]
    n = len(live)
    src = [p for p in reversed(live) if p >= n]
    dst = [p for p in range(n) if want.refs[p] <= 0]
    to = dict(zip(src, dst))
    want.table = [[to.get(e, e) for e in r] for r in want.table]
    for a, b in zip(src, dst):
        want.refs[b], want.refs[a] = want.refs[a], 0
        for t in pools:
            t[:, b] = t[:, a]
    assert kv.counts[:3].tolist() == [len(src), n, n]
    same(kv, want, pools)
    flags()  # (small pools run out)


def test_pages_bad_entries_are_reported_and_harmless(cuda_lib):
    kv = empty_pool(10, 4, 4, 3)
    kv.reserve(dev([0, 5, 2, -1]))
    assert kv.table.tolist() == [[0, -1, -1], [-1, 1, -1], [2, -1, -1], [-1, -1, -1]]
    kv.fork(dev([0, 4, -2, 0]))  # parents out of range: kept
    assert kv.table.tolist() == [[0, -1, -1], [-1, 1, -1], [2, -1, -1], [0, -1, -1]]
    assert flags() == ["bad_page"] and kv.refs.tolist()[:4] == [2, 1, 1, 0]
    kv.table[2, 0] = 99  # an entry outside the pool counts as missing
    kv.reserve(dev([0, -1, 1, -1]))
    assert flags() == ["bad_page"]
    assert kv.counts[:3].tolist() == [1, 0, 2]
    assert kv.table.tolist()[0][0] == 3 and kv.table.tolist()[2][0] == 4
    kv.reserve(dev([12, -9, 2**31 - 1]))
    assert flags() == ["bad_pos"] and kv.counts[:3].tolist() == [0, 0, 0]
    kv.reserve(dev([0, 0]), dev([4, -1]))
    assert flags() == ["bad_page"] and kv.counts[:3].tolist() == [0, 0, 0]
    before = kv.k.clone()
    counts = dev([3])
    kv.copy_pages(dev([0, 10, -1]), dev([7, 2, 3]), counts)
    want = before.clone()
    want[:, 7] = before[:, 0]
    assert torch.equal(kv.k, want) and flags() == ["bad_page"]
    for n in (0, -5):  # nothing to copy
        kv.copy_pages(dev([1]), dev([2]), dev([n]))
        assert torch.equal(kv.k, want)
    kv.copy_pages(dev([1]), dev([8]), dev([1000]))  # a count past the list: the list's length holds
    want[:, 8] = want[:, 1]
    assert torch.equal(kv.k, want) and flags() == []


def test_positions_next_to_the_end_of_32_bits(cuda_lib, rng):
    """Tables that reach past 2^31 positions: the last positions are refused by every call, those before them are not,
    and the other rows of the call are as they are without them."""
    import ctypes

    import gsdlq_b200._lib as L
    from gsdlq_b200 import ops, paged
    page, top = 1 << 30, 2**31 - 129
    table, refs = dev([[-1] * 3, [-1] * 3]), dev([0] * 4)
    desc = L.PagedKVDesc(kv_type=0, layers=1, n_pages=4, page_size=page, n_kv_heads=1, head_dim=32,
                         table=table.data_ptr(), refs=refs.data_ptr(), n_seqs=2, max_blocks=3)  # (no pool is looked at)
    src, dst, counts = dev([-1] * 4), dev([-1] * 4), dev([0] * 4)

    def reserve(pos):
        p = dev(pos)
        assert cuda_lib.gsdlq_pages_reserve(ctypes.byref(desc), None, p.data_ptr(), 2, src.data_ptr(), dst.data_ptr(), 2,
                                            counts.data_ptr(), ops._stream_on(p.device)) == 0
        return counts[:3].tolist()

    assert reserve([top, 5]) == [0, 0, 2] and table.tolist() == [[-1, 0, -1], [1, -1, -1]] and flags() == []
    assert reserve([2**31 - 1, top + 1]) == [0, 0, 0] and flags() == ["bad_pos"]
    # a table of 2^31 + 64 positions over a small pool
    small = make_pool(rng, [40], 16, 1, 64, torch.float16)
    table = torch.full((1, (1 << 27) + 4), -1, dtype=torch.int32, device="cuda")
    table[0, :3] = small.table[0, :3]
    kv = paged.PagedKV.wrap(small.k, small.v, table, small.refs)
    rows = [39, 2**31 - 1, top + 1, 7]
    for pos in (rows, rows[1:] + rows[:1]):
        q = torch.from_numpy(rng.standard_normal((len(pos), 2, 64))).float().cuda()
        got = run_attention(kv, 0, q, pos, [0] * len(pos))
        assert flags() == ["bad_pos"]
        for r, p in enumerate(pos):
            if p > top:
                assert not got[r].any()
                continue
            k, v = rows_of(kv, 0, 0, p + 1)
            want, tol = O.attention(q[r].cpu().numpy(), k, v, 0.125)
            assert (np.abs(got[r] - want) <= tol).all()
    with pytest.raises(L.GsdlqError, match="unsupported"):  # (enough rows to share tiles are too many for such a table)
        run_attention(kv, 0, torch.zeros(128, 2, 64, device="cuda"), rows * 32, [0] * 128)
    cs = torch.zeros(64, 32, 2, device="cuda")
    before = kv.k.clone()
    x = torch.ones(1, 2, 64, device="cuda")
    out = torch.zeros_like(x)
    ops.rope_kv_paged(ops.paged_append_job(kv, 0, x, x[:, :1], x[:, :1], out, dev([2**31 - 1]), cs))
    assert torch.equal(out, x) and torch.equal(kv.k.view(torch.int16), before.view(torch.int16))
    assert flags() == ["bad_pos"]


def test_resized_pool(cuda_lib):
    kv = empty_pool(12, 4, 3, 3)
    kv.reserve(dev([0, 4, 8]))
    kv.reserve(dev([0, 0, 0]))
    kv.fork(dev([-1, 1, 2]))
    with pytest.raises(ValueError):
        kv.resized(3)
    kv.compact()
    n = kv.pages_in_use()
    assert kv.counts[:3].tolist() == [1, n, n]
    small = kv.resized(n)
    assert torch.equal(small.k, kv.k[:, :n]) and torch.equal(small.v, kv.v[:, :n]) and small.n_pages == n
    assert torch.equal(small.refs, kv.refs[:n]) and small.table is kv.table
    big = small.resized(30)
    assert torch.equal(big.k[:, :n], small.k) and big.refs.tolist() == small.refs.tolist() + [0] * (30 - n)
    big.reserve(dev([0, -1, -1]))
    assert big.table[0, 0] == n and flags() == []


# ---------------------------------------------------------------------------------------- as they are used
def test_steps_captured_in_graphs_on_two_streams(cuda_lib, rng):
    """Reserve, append and attention captured and replayed, two caches with a work area each on two streams at
    once, against the eager calls on the default stream."""
    from gsdlq_b200 import ops, paged
    heads, nkv, hd, page, seqs = 8, 2, 64, 4, 3
    cs = torch.from_numpy(rng.standard_normal((64, hd // 2, 2))).float().cuda()

    def setup(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        kv = paged.PagedKV(1, 60, page, nkv, hd, seqs, 16)
        kv.k.fill_(math.nan)
        kv.v.fill_(math.nan)
        x = torch.randn(40, seqs, (heads + 2 * nkv), hd, generator=g, device="cuda")
        cur, pos = x[0].clone(), dev([0, -1, 0])
        out = torch.zeros(seqs, heads, hd, device="cuda")
        q = torch.zeros(seqs, heads, hd, device="cuda")
        append = ops.paged_append_job(kv, 0, cur[:, :heads], cur[:, heads:heads + nkv], cur[:, heads + nkv:], q, pos, cs)
        attn = ops.paged_attn_job(kv, 0, q, out, pos, 0.125, ops.attention_paged_work(kv, seqs, heads))

        def step():
            kv.reserve(pos)
            ops.rope_kv_paged(append)
            ops.attention_paged(attn)
            pos.add_((pos >= 0).int())
        return kv, x, cur, pos, out, step

    steps = 30
    plain = []
    for seed in (1, 2):
        kv, x, cur, pos, out, step = setup(seed)
        res = []
        for i in range(steps):
            cur.copy_(x[i])
            step()
            res.append(out.clone())
        plain.append((torch.stack(res), kv.table.clone(), kv.refs.clone()))
    runs = []
    for seed in (1, 2):
        kv, x, cur, pos, out, step = setup(seed)
        torch.cuda.synchronize()
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            step()  # warm-up; its position is taken back
            pos.sub_((pos >= 0).int())
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=st):
                step()
        runs.append((kv, x, cur, out, g, st, []))
    torch.cuda.synchronize()
    for i in range(steps):
        for kv, x, cur, out, g, st, res in runs:
            with torch.cuda.stream(st):
                cur.copy_(x[i])
                g.replay()
                res.append(out.clone())
    torch.cuda.synchronize()
    for (want, table, refs), (kv, _, _, _, _, _, res) in zip(plain, runs):
        assert torch.equal(torch.stack(res), want)
        assert torch.equal(kv.table, table) and torch.equal(kv.refs, refs)
    assert flags() == []


def test_fork_then_write_keeps_the_others_rows(cuda_lib, rng):
    """Fork, reserve, append, attention: each copy sees the shared prefix and its own new row."""
    from gsdlq_b200 import ops
    kv = make_pool(rng, [21, 0, 0, 0], 8, 2, 64, torch.float16, spare=8, max_blocks=5)
    kv.fork(dev([0, 0, 0, -1]))
    kv.reserve(dev([21, 21, 21, -1]))
    assert kv.counts[:3].tolist() == [2, 0, 2]
    old_k, old_v = rows_of(kv, 0, 2, 21)
    append_check(kv, 0, rng, [21, 21, 21, -1], 4)
    last = []
    for s in range(3):
        k, v = rows_of(kv, 0, s, 22)
        assert np.array_equal(k[:21], old_k) and np.array_equal(v[:21], old_v)
        last.append(k[21])
    assert not np.array_equal(last[0], last[1]) and not np.array_equal(last[1], last[2])
    q = torch.from_numpy(rng.standard_normal((4, 4, 64))).float().cuda()
    check_attention(kv, 0, q, [21, 21, 21, -1])
    kv.fork(dev([-1, -1, -1, -1]))
    assert not kv.refs.any() and (kv.table == -1).all() and flags() == []
