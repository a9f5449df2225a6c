"""Refusals of the paged cache's and the log probabilities' C entry points before any CUDA call (the stand-in
addresses are never dereferenced), the Python checks that need no GPU, and the tests' own restatement of the page
bookkeeping on cases worked out by hand."""
import ctypes
import math

import pytest

import paged_oracle as O
from gsdlq_b200 import _lib as L

torch = pytest.importorskip("torch")

A, ODD4, ODD2 = 0x100000, 0x100004, 0x100002


def kv(**over):
    d = dict(k=A, v=A, kv_type=0, layers=2, n_pages=10, page_size=16, n_kv_heads=2, head_dim=64, table=A, refs=A,
             n_seqs=4, max_blocks=5)
    d.update(over)
    return L.PagedKVDesc(**d)


BAD_PAGES = [dict(n_pages=0), dict(n_pages=(1 << 28) + 1), dict(page_size=0), dict(max_blocks=0), dict(n_seqs=0),
             dict(n_seqs=1025), dict(table=None), dict(refs=None)]
BAD_POOL = BAD_PAGES + [dict(k=None), dict(v=None), dict(k=ODD4), dict(v=ODD4), dict(layers=0), dict(n_kv_heads=0),
                        dict(kv_type=2), dict(kv_type=-1), dict(head_dim=96), dict(head_dim=256), dict(head_dim=0)]


def test_append_refusals():
    lib = L.load()

    def call(pool=None, **over):
        d = dict(layer=1, q=A, k=A, v=A, q_out=A, q_stride=0, kv_stride=0, q_out_stride=0, rope_cs=A, max_pos=80,
                 interleaved=1, row_seq=None, pos=A, rows=4, n_heads=4)
        d.update(over)
        return lib.gsdlq_rope_kv_paged(ctypes.byref(L.PagedAppendJob(kv=kv(**(pool or {})), **d)), None)

    assert lib.gsdlq_rope_kv_paged(None, None) == -1
    for bad in BAD_POOL:
        assert call(bad) == -1, bad
    for bad in (dict(layer=-1), dict(layer=2), dict(q=None), dict(k=None), dict(v=None), dict(q_out=None),
                dict(rope_cs=None), dict(max_pos=0), dict(pos=None), dict(rows=0), dict(rows=5), dict(n_heads=0),
                dict(q_stride=255), dict(q_stride=-1), dict(q_out_stride=255), dict(kv_stride=127),
                dict(q_stride=300), dict(n_heads=1 << 30)):
        assert call(**bad) == -1, bad


def test_attention_refusals():
    lib = L.load()
    n = ctypes.c_size_t()
    assert lib.gsdlq_attention_paged_work_size(4, 8, 2, 64, ctypes.byref(n)) == 0
    ok = n.value
    assert ok % 16 == 0 and ok > 4 * 4 * 2
    for bad in ((0, 8, 2, 64), (4, 0, 2, 64), (4, 8, 0, 64), (4, 7, 2, 64), (4, 8, 2, 96), (-1, 8, 2, 64)):
        assert lib.gsdlq_attention_paged_work_size(*bad, ctypes.byref(n)) == -1, bad
    assert lib.gsdlq_attention_paged_work_size(4, 8, 2, 64, None) == -1

    def call(pool=None, **over):
        d = dict(layer=1, q=A, q_stride=0, out=A, row_seq=None, pos=A, rows=4, n_heads=8, sm_scale=0.125, work=A,
                 work_bytes=ok)
        d.update(over)
        return lib.gsdlq_attention_paged(ctypes.byref(L.PagedAttnJob(kv=kv(**(pool or {})), **d)), None)

    assert lib.gsdlq_attention_paged(None, None) == -1
    for bad in BAD_POOL:
        assert call(bad) == -1, bad
    for bad in (dict(layer=-1), dict(layer=2), dict(q=None), dict(q=ODD4), dict(q_stride=514), dict(q_stride=508),
                dict(q_stride=-4), dict(out=None), dict(out=ODD4), dict(pos=None), dict(rows=0), dict(rows=5),
                dict(n_heads=7), dict(n_heads=0), dict(work=None), dict(work=ODD4), dict(work_bytes=ok - 1)):
        assert call(**bad) == -1, bad
    # places or units past 31 bits: refused as unsupported, before any CUDA call
    assert call(dict(n_pages=1 << 27, page_size=16)) == -3
    assert call(dict(page_size=1 << 10, max_blocks=1 << 24), work_bytes=ok) == -3


def test_page_refusals():
    lib = L.load()
    d = ctypes.byref
    assert lib.gsdlq_pages_fork(None, A, None) == -1 and lib.gsdlq_pages_fork(d(kv()), None, None) == -1
    for bad in BAD_PAGES:
        assert lib.gsdlq_pages_fork(d(kv(**bad)), A, None) == -1, bad
        assert lib.gsdlq_pages_reserve(d(kv(**bad)), None, A, 4, A, A, 4, A, None) == -1, bad
        assert lib.gsdlq_pages_compact(d(kv(**bad)), A, A, 4, A, A, 1 << 31, None) == -1, bad
    for bad in BAD_POOL:
        assert lib.gsdlq_pages_copy(d(kv(**bad)), A, A, A, 4, None) == -1, bad

    def reserve(seq=None, pos=A, rows=4, src=A, dst=A, most=4, counts=A):
        return lib.gsdlq_pages_reserve(d(kv()), seq, pos, rows, src, dst, most, counts, None)

    for bad in (dict(pos=None), dict(rows=0), dict(rows=5, most=9), dict(seq=A, rows=1025, most=2000), dict(src=None),
                dict(dst=None), dict(most=3), dict(counts=None)):
        assert reserve(**bad) == -1, bad

    def compact(src=A, dst=A, most=4, counts=A, work=A, wb=40):
        return lib.gsdlq_pages_compact(d(kv()), src, dst, most, counts, work, wb, None)

    for bad in (dict(src=None), dict(dst=None), dict(most=0), dict(counts=None), dict(work=None), dict(work=ODD2),
                dict(wb=39)):
        assert compact(**bad) == -1, bad
    for bad in ((None, A, A, 4), (A, None, A, 4), (A, A, None, 4), (A, A, A, 0), (A, A, A, -1)):
        assert lib.gsdlq_pages_copy(d(kv()), *bad, None) == -1, bad


def test_logprobs_refusals():
    lib = L.load()

    def call(**over):
        d = dict(logits=A, row_stride=0, rows=2, n=100, temperature=1.0, ids=A, logprob=A, entropy=A, top=5, top_ids=A,
                 top_logprobs=A)
        d.update(over)
        return lib.gsdlq_logprobs_rows(ctypes.byref(L.LogprobsJob(**d)), None)

    assert lib.gsdlq_logprobs_rows(None, None) == -1
    for bad in (dict(logits=None), dict(rows=0), dict(n=0), dict(row_stride=99), dict(temperature=0.0),
                dict(temperature=-1.0), dict(temperature=math.inf), dict(temperature=math.nan), dict(ids=None),
                dict(logprob=None), dict(top=-1), dict(top=33), dict(top=5, n=4), dict(top_ids=None),
                dict(top_logprobs=None), dict(ids=None, logprob=None, entropy=None, top=0), dict(logits=ODD2)):
        assert call(**bad) == -1, bad


def test_tensors_off_the_gpu_are_refused():
    from gsdlq_b200 import ops, paged
    t = dict(dtype=torch.int32)
    k = torch.zeros(1, 4, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA device"):
        paged.PagedKV.wrap(k, k.clone(), torch.zeros(2, 3, **t), torch.zeros(4, **t))
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        paged.PagedKV.wrap(k.float(), k.float(), torch.zeros(2, 3, **t), torch.zeros(4, **t))
    with pytest.raises(TypeError, match="must be a tensor"):
        paged.PagedKV.wrap(k, None, torch.zeros(2, 3, **t), torch.zeros(4, **t))
    with pytest.raises(ValueError, match="at least 1"):
        paged.PagedKV(1, 0, 16, 2, 64, 2, 3, device="cpu")
    with pytest.raises(ValueError, match="CUDA device"):
        ops.logprobs_job(torch.zeros(2, 10), entropy=torch.zeros(2))
    with pytest.raises(TypeError):
        ops.logprobs_job([[0.0]], entropy=torch.zeros(1))


def test_launches_stay_on_the_current_device(monkeypatch):
    """A launch goes to the current device's stream, so tensors on another device are refused."""
    from gsdlq_b200 import ops
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="cuda:0 is the current device"):
        ops._stream_on(torch.device("cuda", 1))


def test_struct_sizes_match_the_header(tmp_path):
    """The ctypes structs have the C structs' sizes."""
    import os
    import shutil
    import subprocess
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "gsdlq.h"\nint main(void) { printf("%zu %zu %zu %zu", '
                   "sizeof(gsdlq_paged_kv_t), sizeof(gsdlq_paged_append_job_t), sizeof(gsdlq_paged_attn_job_t), "
                   "sizeof(gsdlq_logprobs_job_t)); return 0; }\n")
    exe = tmp_path / "sizes"
    subprocess.run([cc, "-std=c99", "-I", os.path.dirname(L.HEADER), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(t) for t in (L.PagedKVDesc, L.PagedAppendJob, L.PagedAttnJob, L.LogprobsJob)]


def test_restated_page_bookkeeping():
    p = O.Pages([[-1] * 3 for _ in range(4)], [0] * 6, 4)
    assert p.reserve([(0, 0), (0, 3), (0, 4), (2, -1), (1, 9)]) == ([], 0, 3)
    assert p.table == [[0, 1, -1], [-1, -1, 2], [-1] * 3, [-1] * 3] and p.refs == [1, 1, 1, 0, 0, 0]
    p.fork([0, 0, 0, -1])                        # 1 drops page 2 and shares 0's, so does 2
    assert p.table[:3] == [[0, 1, -1]] * 3 and p.refs == [3, 3, 0, 0, 0, 0]
    assert p.reserve([(0, 5), (1, 5), (2, 5)]) == ([(1, 2), (1, 3)], 0, 2)  # the last holder keeps page 1
    assert [r[1] for r in p.table[:3]] == [2, 3, 1] and p.refs == [3, 1, 1, 1, 0, 0]
    assert p.reserve([(0, 0), (1, 0), (2, 0), (2, 8)]) == ([(0, 4), (0, 5)], 1, 2)
    assert p.reserve([(0, 8), (1, 8)]) == ([], 2, 0)
    p.fork([-1, 1, 2, 3])
    assert p.refs == [1, 1, 0, 1, 0, 1]
    assert p.compact(1) == ([(5, 2)], 4, 4) and p.table[1][0] == 2
    assert p.compact(9) == ([], 4, 4)


def test_attention_work_serves_every_shape_in_turn():
    """What a launch keeps beside its counters has one size whatever its shape is, so that one area serves launches of
    any rows, heads and head sizes in turn."""
    lib = L.load()

    def size(rows, heads, kv_heads, hd):
        n = ctypes.c_size_t()
        assert lib.gsdlq_attention_paged_work_size(rows, heads, kv_heads, hd, ctypes.byref(n)) == 0
        return n.value

    for rows, heads, kv_heads in ((1, 4, 4), (128, 32, 32), (300, 32, 8), (7, 40, 2)):
        items = rows * kv_heads * -(-heads // kv_heads // 8)  # groups of up to eight heads
        assert len({size(rows, heads, kv_heads, hd) - -(-items // 4) * 16 for hd in (32, 64, 128)}) == 1
    parts = {size(rows, heads, kv_heads, hd) - -(-rows * kv_heads // 4) * 16
             for rows, heads, kv_heads, hd in ((1, 4, 4, 32), (128, 32, 32, 64), (300, 32, 8, 128), (2, 2, 1, 64))}
    assert len(parts) == 1
    assert all(size(r, 32, 8, 64) <= size(r + 1, 32, 8, 64) for r in range(1, 70))


def test_append_refuses_angles_off_their_pairs():
    """The angles are read in pairs, so a table that starts at an odd element is refused before any launch."""
    lib = L.load()
    for off in (4, 12, 1):
        job = L.PagedAppendJob(kv=kv(), layer=1, q=A, k=A, v=A, q_out=A, rope_cs=A + off, max_pos=80, interleaved=1, pos=A,
                               rows=4, n_heads=4)
        assert lib.gsdlq_rope_kv_paged(ctypes.byref(job), None) == -1


def test_refused_generations_leave_the_sequences_alone():
    import types

    from gsdlq_b200.paged import PagedBatchDecoder
    d = PagedBatchDecoder.__new__(PagedBatchDecoder)
    d.m, d.B, d.S = types.SimpleNamespace(vocab_size=100), 2, 64
    table, refs = torch.full((2, 4), -1, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    d.kv = types.SimpleNamespace(n_pages=6, page_size=16, table=table, refs=refs)

    def touched(*a, **k):
        raise AssertionError("the sequences were touched")

    d.free = d.fork = d.prefill = d.set_tokens = touched
    for prompts, n, error in (([[1]], 2, ValueError), ([[1], []], 2, ValueError), ([[1], [2] * 60], 5, ValueError),
                              ([[1], [2, 100]], 2, ValueError), ([[1] * 40, [2] * 49], 10, MemoryError)):
        with pytest.raises(error):
            d.generate(prompts, n)
    for prompt, beams, n, error in (([], 2, 4, ValueError), ([1], 3, 4, ValueError), ([1], 2, 64, ValueError),
                                    ([1], 2, 0, ValueError), ([5, -1], 2, 4, ValueError), ([1], 2, 60, MemoryError)):
        with pytest.raises(error):
            d.beam_search(prompt, beams, n)
    with pytest.raises(AssertionError):
        d.generate([[1], [2]], 3)


def test_row_strides_past_an_int_are_refused():
    """The row descriptors hold strides as ints: a wider one must not be cut off."""
    from gsdlq_b200 import ops
    t = lambda stride: torch.empty_strided((2, 4), (stride, 1), device="meta")  # noqa: E731
    assert ops._row_stride(t(2**31 - 1)) == 2**31 - 1 and ops._row_stride(t(2**40)[:1]) == 0
    for stride in (2**31, 2**32 + 256):
        with pytest.raises(ValueError, match="apart"):
            ops._row_stride(t(stride))
    assert ops._row_stride(t(2**32), 2**63 - 1) == 2**32  # (that of logits is a size_t)


def test_attention_refuses_a_scale_that_is_not_finite():
    """From C too, and where a Python float is past the descriptor's fp32."""
    lib = L.load()
    n = ctypes.c_size_t()
    assert lib.gsdlq_attention_paged_work_size(4, 8, 2, 64, ctypes.byref(n)) == 0
    for scale in (math.nan, math.inf, -math.inf, 1e39):
        job = L.PagedAttnJob(kv=kv(), layer=1, q=A, out=A, pos=A, rows=4, n_heads=8, sm_scale=scale, work=A, work_bytes=n.value)
        assert lib.gsdlq_attention_paged(ctypes.byref(job), None) == -1


def test_generations_leave_room_for_other_tables_pages():
    """Pages that this decoder's own table names are free for a generation; those that others over the pool hold are
    not, also where this one names them too."""
    import types

    from gsdlq_b200.paged import PagedBatchDecoder
    d = PagedBatchDecoder.__new__(PagedBatchDecoder)
    d.m, d.B, d.S = types.SimpleNamespace(vocab_size=100), 2, 64
    table = torch.tensor([[0, 1, -1, -1], [0, 3, 99, -1]], dtype=torch.int32)

    def room(refs, pages):
        d.kv = types.SimpleNamespace(n_pages=6, page_size=16, table=table, refs=torch.tensor(refs, dtype=torch.int32))
        d._room([pages * 16])

    for refs, have in (([2, 1, 0, 1, 0, 0], 6), ([2, 1, 1, 1, 0, 0], 5), ([3, 1, 1, 2, 0, 4], 2)):
        room(refs, have)
        with pytest.raises(MemoryError, match=f"{have} free"):
            room(refs, have + 1)
