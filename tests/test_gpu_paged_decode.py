"""The paged operators as the engine uses them: PagedBatchDecoder against BatchDecoder and the batch-1 engine,
shared prompts, beam search against its definition, and scoring of a sequence.

Two ways through the engine give logits that agree within LOGIT_TOL (the dequant-GEMM adds with atomics, so the
last bits differ from run to run); picks may differ only at near-ties."""
import math

import numpy as np
import pytest

from conftest import NEAR_TIE, top2_margin

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LOGIT_TOL = 1e-2


def model(name, mode, max_seq=320, **over):
    import gsdlq_b200.packer as P
    from gsdlq_b200.model import GSDLQModel
    cfg = P.make_config(name, **over)
    return GSDLQModel(P.random_model_cuda(cfg, mode, seed=31, norm_jitter=0.1), max_seq=max_seq), cfg


def log_softmax(x):
    x = np.asarray(x, np.float64)
    x = x - x.max(-1, keepdims=True)
    return x - np.log(np.exp(x).sum(-1, keepdims=True))


@pytest.mark.parametrize("name,mode,batch,page,dtype", [
    ("smollm2-1.7b", "turbo", 6, 16, torch.float16),
    ("mistral-7b", "precision", 4, 24, torch.float16),
    ("qwen2.5-1.5b", "precision", 3, 64, torch.bfloat16),
])
def test_paged_decode_matches_the_contiguous_cache(cuda_lib, name, mode, batch, page, dtype):
    import gsdlq_b200._lib as L
    from gsdlq_b200.batch import BatchDecoder
    from gsdlq_b200.paged import PagedBatchDecoder
    m, cfg = model(name, mode, n_layers=2)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, cfg["vocab_size"], int(n)).tolist() for n in rng.integers(2, 200, batch)]
    prompts[0] = prompts[0][:1]
    bd = BatchDecoder(m, batch, max_seq=320)
    pages = sum(-(-(len(p) + 8) // page) for p in prompts)
    pd = PagedBatchDecoder(m, batch, pages, page, max_seq=320, kv_dtype=dtype)
    for b, pr in enumerate(prompts):
        bd.prefill(b, pr[:-1])
        pd.prefill(b, pr[:-1])
    at = [len(pr) - 1 for pr in prompts]
    bd.set_tokens([pr[-1] for pr in prompts], at)
    pd.set_tokens([pr[-1] for pr in prompts], at)
    tol = LOGIT_TOL if dtype == torch.float16 else 0.2  # a bf16 cache: 2^-9 per stored value instead of 2^-12
    for step in range(8):
        bd.step()
        pd.step()
        a, b = bd.logits_host(), pd.logits_host()
        assert np.abs(a - b).max() < tol
        pa, pb = bd.ids.cpu().numpy(), pd.ids.cpu().numpy()
        for s in np.flatnonzero(pa != pb):
            assert top2_margin(a[s]) < max(NEAR_TIE, 2 * tol * (dtype != torch.float16))
        pd.ids.copy_(bd.ids)
        assert torch.equal(bd.pos, pd.pos)
    lp = pd.logprobs(top=4)
    want = log_softmax(pd.logits_host())
    assert np.abs(lp["top_logprobs"] - -np.sort(-want, 1)[:, :4]).max() < 1e-4
    assert np.array_equal(lp["top_ids"][:, 0], pd.logits_host().argmax(1))
    assert L.device_flags() == 0 and pd.kv.pages_in_use() <= pages
    bd.release()
    pd.release()
    m.release()


@pytest.mark.parametrize("batch", [2, 16, 32, 128])
def test_prompts_between_steps_match_the_contiguous_cache(cuda_lib, batch):
    """One decoder takes prompts and steps in turn: chunks of 128 rows and fewer and steps of ``batch`` rows follow one
    another in every order, and each step's logits are those of the contiguous cache."""
    import gsdlq_b200._lib as L
    from gsdlq_b200.batch import BatchDecoder
    from gsdlq_b200.paged import PagedBatchDecoder
    m, cfg = model("smollm2-1.7b", "turbo", n_layers=2)
    rng = np.random.default_rng(17)
    vocab, S = cfg["vocab_size"], 320
    bd = BatchDecoder(m, batch, max_seq=S)
    pd = PagedBatchDecoder(m, batch, batch * 20, 16, max_seq=S)
    at, tok = [0] * batch, rng.integers(0, vocab, batch).tolist()

    def prompt(b, n):
        ids = rng.integers(0, vocab, n).tolist()
        for d in (bd, pd):
            d.prefill(b, ids[:-1])
        at[b], tok[b] = n - 1, ids[-1]

    def steps(n):
        for d in (bd, pd):
            d.set_tokens(tok, at)
        for _ in range(n):
            bd.step()
            pd.step()
            a, b = bd.logits_host(), pd.logits_host()
            assert np.abs(a - b).max() < LOGIT_TOL
            pd.ids.copy_(bd.ids)
            for s in range(batch):
                at[s] += 1
        tok[:] = bd.ids.tolist()

    prompt(0, 150)
    prompt(1, 300)
    steps(2)
    for b, n in ((0, 300), (1, 130), (batch - 1, 290), (0, 3)):
        pd.free([b])
        prompt(b, n)
        steps(2)
    pd.free(range(batch))
    for b in range(batch):
        prompt(b, int(rng.integers(2, 310)))
    steps(3)
    assert L.device_flags() == 0
    bd.release()
    pd.release()
    m.release()


def test_generate_idle_sequences_and_page_exhaustion(cuda_lib):
    import gsdlq_b200._lib as L
    from gsdlq_b200.paged import PagedBatchDecoder
    m, cfg = model("smollm2-1.7b", "turbo", n_layers=1)
    rng = np.random.default_rng(5)
    pd = PagedBatchDecoder(m, 4, 24, 16, max_seq=320)
    prompts = [rng.integers(0, cfg["vocab_size"], n).tolist() for n in (40, 3, 16, 17)]
    a = pd.generate(prompts, 12)
    assert [len(x) for x in a] == [12] * 4
    # sequences 1 and 3 idle: the others go on alike, the idle ones hold no pages
    pd.free([1, 3])
    used = pd.kv.pages_in_use()
    assert pd.pos.tolist()[1] == -1 == pd.pos.tolist()[3] and pd.pos.tolist()[0] == 51
    for _ in range(3):
        pd.step()
    assert pd.pos.tolist() == [54, -1, 30, -1] and pd.kv.pages_in_use() == used
    n = pd.compact()
    assert n == used and pd.kv.counts[2] == n
    with pytest.raises(MemoryError):
        pd.generate([list(range(100))] * 4, 100)
    assert L.device_flags() == 0
    # no host check on single steps: a step that finds no page reports it and leaves other sequences' rows alone
    pd.free(range(4))
    with pytest.raises(MemoryError):
        for b in range(3):
            pd.prefill(b, rng.integers(0, cfg["vocab_size"], 190).tolist())
    assert L.flag_names(L.device_flags()) == ["no_page"]
    pd.free(range(4))
    for b in range(2):
        pd.prefill(b, rng.integers(0, cfg["vocab_size"], 190).tolist())
    before = pd.kv.k.clone()
    pd.set_tokens([1, 2, 3, 4], [190, 190, 0, 0])
    pd.step()
    assert set(L.flag_names(L.device_flags())) == {"no_page", "bad_page"}
    table = pd.kv.table[0, :11].long()
    assert torch.equal(before[:, table], pd.kv.k[:, table])
    for bad in (lambda: pd.set_tokens([1] * 4, [-2, 0, 0, 0]), lambda: pd.set_tokens([1] * 3, [0] * 4),
                lambda: pd.prefill(4, [1]), lambda: pd.prefill(0, [1], 320), lambda: pd.fork([0, 1, 2, 4]),
                lambda: pd.fork([0, 1]), lambda: pd.free([4]), lambda: pd.generate(prompts[:2], 2),
                lambda: pd.beam_search([], 2, 4), lambda: pd.beam_search([1], 5, 4), lambda: pd.beam_search([1], 2, 400)):
        with pytest.raises(ValueError):
            bad()
    pd.release()
    m.release()


def test_shared_prompt_continues_like_separate_prefills(cuda_lib):
    """One prefill forked into three continuations with tokens of their own, against the batch-1 engine on each."""
    import gsdlq_b200._lib as L
    from gsdlq_b200.paged import PagedBatchDecoder
    m, cfg = model("mistral-7b", "precision", n_layers=2)
    rng = np.random.default_rng(9)
    prompt = rng.integers(0, cfg["vocab_size"], 150).tolist()
    toks = rng.integers(0, cfg["vocab_size"], (4, 3)).tolist()
    pd = PagedBatchDecoder(m, 3, 30, 16, max_seq=320)
    pd.prefill(0, prompt)
    pages = pd.kv.pages_in_use()
    pd.fork([0, 0, 0])
    assert pd.kv.pages_in_use() == pages
    got = []
    for i, t in enumerate(toks):
        pd.set_tokens(t, [len(prompt) + i] * 3)
        pd.step_logits()
        got.append(pd.logits_host())
    assert pd.kv.pages_in_use() == pages + 2  # the last, partly filled page: one copy for all but the last holder
    for s in range(3):
        m.prefill(prompt)
        for i, t in enumerate(toks):
            lg = m.forward_token(t[s], len(prompt) + i)
            assert np.abs(lg - got[i][s]).max() < LOGIT_TOL
    assert L.device_flags() == 0
    pd.release()
    m.release()


def test_beam_search_follows_its_definition(cuda_lib):
    """Against a beam search on the host over the batch-1 engine's logits.  Where the order of two candidates at
    the beam's edge hangs on less than the logits' tolerance the searches may part: the sums still agree within
    the tolerance per step."""
    import gsdlq_b200._lib as L
    from gsdlq_b200.paged import PagedBatchDecoder
    m, cfg = model("smollm2-1.7b", "turbo", n_layers=2)
    rng = np.random.default_rng(11)
    prompt = rng.integers(0, cfg["vocab_size"], 37).tolist()
    beams, steps = 3, 5
    pd = PagedBatchDecoder(m, 4, 24, 16, max_seq=320)
    for eos in (None, "second"):
        live, done = [([], 0.0)], []
        for i in range(steps):
            cand = []
            for toks, s in live:
                m.prefill((prompt + toks)[:-1])
                lp = log_softmax(m.forward_token((prompt + toks)[-1], len(prompt + toks) - 1))
                if eos == "second":
                    eos = int(np.argsort(-lp)[1])
                cand += [(s + lp[t], toks + [int(t)]) for t in np.argsort(-lp)[:beams + 2]]
            cand.sort(key=lambda c: -c[0])
            live = []
            for s, toks in cand:
                if len(live) < beams:
                    if toks[-1] == eos:
                        done.append((toks[:-1], s))
                    else:
                        live.append((toks, s))
            done = sorted(done, key=lambda d: -d[1])[:beams]
            if len(done) == beams and done[-1][1] >= live[0][1]:
                break
        want = sorted(done + live, key=lambda d: -d[1])[:beams]
        got = pd.beam_search(prompt, beams, steps, eos)
        assert len(got) == beams
        assert np.allclose([s for _, s in got], [s for _, s in want], atol=2 * steps * LOGIT_TOL)
        gaps = np.diff([s for _, s in want])
        if (np.abs(gaps) > 4 * steps * LOGIT_TOL).all():
            assert [t for t, _ in got] == [t for t, _ in want]
    # greedy is beam search with one beam
    one = pd.beam_search(prompt, 1, 4)[0][0]
    lg = None
    m.prefill(prompt[:-1])
    for i, t in enumerate([prompt[-1]] + one[:-1]):
        lg = m.forward_token(t, len(prompt) - 1 + i)
        assert one[i] == int(np.argmax(lg)) or top2_margin(lg) < NEAR_TIE
    assert L.device_flags() == 0
    pd.release()
    m.release()


def test_score_matches_the_token_by_token_logits(cuda_lib):
    import gsdlq_b200._lib as L
    m, cfg = model("qwen2.5-1.5b", "precision", n_layers=2)
    rng = np.random.default_rng(13)
    ids = rng.integers(0, cfg["vocab_size"], 131).tolist()  # one chunk and a bit
    got = m.score(ids, top=3)
    assert got["logprob"].shape == (131,) and got["top_ids"].shape == (131, 3) and got["logprob"][-1] == 0.0
    for i, t in enumerate(ids):
        if i in (0, 1, 64, 127, 128, 129, 130):
            lp = log_softmax(m.forward_token(t, i))
            if i + 1 < len(ids):
                assert abs(got["logprob"][i] - lp[ids[i + 1]]) < 2 * LOGIT_TOL
            assert abs(got["entropy"][i] + (np.exp(lp) * lp).sum()) < 0.1
            assert np.abs(got["top_logprobs"][i] - np.sort(lp)[::-1][:3]).max() < 2 * LOGIT_TOL
    last = m.logprobs([5], top=2)
    lp = log_softmax(m.logits_host())
    assert abs(last["logprob"][0] - lp[5]) < 1e-4 and last["top_ids"][0, 0] == int(np.argmax(lp))
    assert m.score(ids[:1])["logprob"].tolist() == [0.0]
    for bad in ([], [cfg["vocab_size"]], [-1], [0] * 321):
        with pytest.raises(ValueError):
            m.score(bad)
    with pytest.raises(ValueError):
        m.logprobs([1, 2])
    with pytest.raises(ValueError):
        m.logprobs(top=33)
    assert L.device_flags() == 0
    m.release()


def test_wrong_tensors_are_refused(cuda_lib):
    from gsdlq_b200 import ops, paged
    kv = paged.PagedKV(2, 8, 16, 2, 64, 3, 4)
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    q, k, cs, pos = f(3, 4, 64), f(3, 2, 64), f(64, 32, 2), i(3)
    work = ops.attention_paged_work(kv, 3, 4)
    ops.paged_append_job(kv, 0, q, k, k, q, pos, cs)
    ops.paged_attn_job(kv, 0, q, f(3, 4, 64), pos, 0.125, work)
    bad = [
        lambda: ops.paged_append_job(kv, 2, q, k, k, q, pos, cs), lambda: ops.paged_append_job(kv, 0, q.half(), k, k, q, pos, cs),
        lambda: ops.paged_append_job(kv, 0, q, f(3, 2, 32), k, q, pos, cs),
        lambda: ops.paged_append_job(kv, 0, q, k, f(3, 4, 64)[:, :2], q, pos, cs),
        lambda: ops.paged_append_job(kv, 0, q, k, k, q, pos.long(), cs),
        lambda: ops.paged_append_job(kv, 0, q, k, k, q, pos.cpu(), cs),
        lambda: ops.paged_append_job(kv, 0, f(4, 4, 64), f(4, 2, 64), f(4, 2, 64), f(4, 4, 64), i(4), cs),
        lambda: ops.paged_append_job(kv, 0, q.expand(3, 4, 64).transpose(0, 1), k, k, q, pos, cs),
        lambda: ops.paged_append_job(kv, 0, f(1, 4, 64).expand(3, 4, 64), k, k, q, pos, cs),
        lambda: ops.paged_append_job(kv, 0, q, k, k, q, pos, f(64, 16, 2)),
        lambda: ops.paged_attn_job(kv, 0, f(3, 3, 64), f(3, 3, 64), pos, 0.125, work),
        lambda: ops.paged_attn_job(kv, 0, q, f(3, 8, 64)[:, ::2], pos, 0.125, work),
        lambda: ops.paged_attn_job(kv, 0, q, f(3, 4, 64), pos, math.nan, work),
        lambda: ops.paged_attn_job(kv, 0, f(3 * 256 + 1)[1:].view(3, 4, 64), f(3, 4, 64), pos, 0.125, work),
        lambda: ops.paged_attn_job(kv, 0, q, f(3, 4, 64), pos, 0.125, work, i(2)),
        lambda: ops.paged_attn_job(kv, -1, q, f(3, 4, 64), pos, 0.125, work),
        lambda: kv.fork(i(2)), lambda: kv.fork(torch.zeros(3, device="cuda")), lambda: kv.reserve(i(4)),
        lambda: kv.reserve(i(2000), i(2000)), lambda: kv.compact(0), lambda: kv.copy_pages(i(2), i(3), i(1)),
        lambda: kv.copy_pages(i(0), i(0), i(1)), lambda: kv.resized(0),
        lambda: paged.PagedKV(1, 4, 16, 2, 96, 1, 1), lambda: paged.PagedKV(1, 4, 16, 2, 64, 1025, 1),
        lambda: paged.PagedKV(1, 4, 16, 2, 64, 1, 1, torch.float32),
        lambda: paged.PagedKV.wrap(kv.k, kv.v[:, :4], kv.table, kv.refs),
        lambda: paged.PagedKV.wrap(kv.k, kv.v, kv.table, kv.refs[:4]),
        lambda: paged.PagedKV.wrap(kv.k.transpose(0, 1), kv.v.transpose(0, 1), kv.table, i(2)),
        lambda: ops.logprobs_job(f(2, 10), entropy=f(3)), lambda: ops.logprobs_job(f(2, 10)),
        lambda: ops.logprobs_job(f(2, 10), ids=i(2)), lambda: ops.logprobs_job(f(2, 10).half(), entropy=f(2)),
        lambda: ops.logprobs_job(f(2, 10), top_ids=i(2, 11), top_logprobs=f(2, 11)),
        lambda: ops.logprobs_job(f(2, 10), entropy=f(2), temperature=0.0),
        lambda: ops.logprobs_job(f(10, 2).t(), entropy=f(2)), lambda: ops.logprobs_job(f(0, 5), entropy=f(0)),
    ]
    for n, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            raise AssertionError(n)
    # a work area too small is refused by the call itself
    small = ops.paged_attn_job(kv, 0, q, f(3, 4, 64), pos, 0.125, work[:64])
    with pytest.raises(Exception, match="invalid argument"):
        ops.attention_paged(small)


def test_angles_off_their_pairs_are_refused(cuda_lib):
    """By the job, so that no launch is made with them."""
    from gsdlq_b200 import ops, paged
    kv = paged.PagedKV(1, 8, 16, 2, 64, 3, 4)
    q, k = torch.zeros(3, 4, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    flat = torch.zeros(64 * 64 + 2, device="cuda")
    ops.paged_append_job(kv, 0, q, k, k, q, pos, flat[2:].view(64, 32, 2))
    with pytest.raises(ValueError, match="rope_cs"):
        ops.paged_append_job(kv, 0, q, k, k, q, pos, flat[1:-1].view(64, 32, 2))


def test_logprobs_are_the_picks_whatever_the_next_inputs_are(cuda_lib):
    """Without token ids: those of the logits' best tokens, after a step, after the next tokens were set, after the
    logits of set tokens without a pick, and after a fork."""
    import gsdlq_b200._lib as L
    from gsdlq_b200.batch import BatchDecoder
    from gsdlq_b200.paged import PagedBatchDecoder
    m, cfg = model("smollm2-1.7b", "turbo", n_layers=1)

    def check(d):
        want = log_softmax(d.logits_host())
        assert np.abs(d.logprobs()["logprob"] - want.max(1)).max() < 1e-4
        own = d.logprobs([7] * d.B)["logprob"]
        assert np.abs(own - want[:, 7]).max() < 1e-4

    for d in (BatchDecoder(m, 3, max_seq=64), PagedBatchDecoder(m, 3, 12, 16, max_seq=64)):
        d.set_tokens([5, 6, 7], [0, 0, 0])
        d.step()
        check(d)
        d.set_tokens([11, 12, 13], [1, 1, 1])
        check(d)
        if isinstance(d, PagedBatchDecoder):
            d.step_logits()
            assert d.ids.tolist() == [11, 12, 13] and d.pos.tolist() == [1, 1, 1]
            check(d)
            d.fork([2, 2, 0])
            check(d)
        d.release()
    assert L.device_flags() == 0
    m.release()


def test_what_just_fits_the_pool_is_not_refused(cuda_lib):
    """20 prompt tokens and 13 new ones store 32 positions, two pages; three beams share the prompt's full page."""
    import gsdlq_b200._lib as L
    from gsdlq_b200.paged import PagedBatchDecoder
    m, cfg = model("smollm2-1.7b", "turbo", n_layers=1)
    rng = np.random.default_rng(23)
    prompts = rng.integers(0, cfg["vocab_size"], (2, 20)).tolist()
    pd = PagedBatchDecoder(m, 2, 4, 16, max_seq=64)
    assert [len(x) for x in pd.generate(prompts, 13)] == [13, 13]
    assert pd.kv.pages_in_use() == 4
    with pytest.raises(MemoryError):
        pd.generate(prompts, 14)
    pd.release()
    for page, pages, n in ((16, 4, 13), (4, 4 + 3 * 4, 13), (1, 19 + 3 * 13, 13)):
        pd = PagedBatchDecoder(m, 3, pages, page, max_seq=64)
        assert [len(t) for t, _ in pd.beam_search(prompts[0], 3, n)] == [n] * 3
        assert pd.kv.pages_in_use() <= pages
        with pytest.raises(MemoryError):
            pd.beam_search(prompts[0], 3, n + 1)
        pd.release()
    assert L.device_flags() == 0
    m.release()


def test_token_ids_of_wider_types_are_not_cut_off(cuda_lib):
    import gsdlq_b200._lib as L
    from gsdlq_b200.model import GSDLQModel
    logits = torch.arange(40.0, device="cuda").reshape(4, 10)
    m = GSDLQModel.__new__(GSDLQModel)
    got = m._logprobs(logits, torch.tensor([2**32 + 5, -1, 9, -2**40 - 1]), 0, 1.0)["logprob"]
    assert got[[0, 1, 3]].tolist() == [0, 0, 0] and abs(got[2] - log_softmax(np.arange(10))[9]) < 1e-5
    assert L.flag_names(L.device_flags()) == ["bad_token"]
    got = m._logprobs(logits, torch.tensor([5, -1, 9, 0]), 0, 1.0)["logprob"]
    assert np.abs(got - log_softmax(np.arange(10))[[5, 0, 9, 0]] * [1, 0, 1, 1]).max() < 1e-5
    assert L.device_flags() == 0
