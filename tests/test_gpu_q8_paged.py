"""The batched grouped-Q8 engine on a paged KV cache: the same logits and token streams as
on the fixed cache, whose oracle and tolerances these tests share (fp32 pages), pages taken,
returned and waited for, and 16-bit pages within what their roundings allow."""
import numpy as np
import pytest

from test_gpu_q8_batch import VOCAB, close, oracle_prompt_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def oracle(oracle_lib, q8_model_bytes):
    return oracle_lib.Q8Oracle(q8_model_bytes)


@pytest.fixture(scope="module")
def paged(native, q8_model_bytes):
    h = native.Q8BatchHandle(0, q8_model_bytes, max_rows=512, slots=6, kv_type="f32", page_size=16)
    yield h
    h.close()


@pytest.mark.parametrize("n", [1, 16, 40, 256])
def test_prefill_logits(paged, oracle, n):
    prompt = np.random.default_rng(n).integers(0, VOCAB, n).tolist()
    close(paged.prefill(0, prompt), oracle_prompt_logits(oracle, prompt))


def test_rows_of_several_slots_and_single_rows(paged, oracle):
    """Ragged rows of two slots, then one row of each: prompt and single-token attention."""
    rng = np.random.default_rng(12)
    p1, p2 = rng.integers(0, VOCAB, 9).tolist(), rng.integers(0, VOCAB, 18).tolist()
    got = paged.forward(p1[:-1] + p2[:-1], list(range(8)) + list(range(17)), [3] * 8 + [5] * 17, [7, 24])
    close(got[0], oracle_prompt_logits(oracle, p1[:-1]))
    close(got[1], oracle_prompt_logits(oracle, p2[:-1]))
    got = paged.forward([p2[-1], p1[-1]], [17, 8], [5, 3], [0, 1])
    close(got[0], oracle_prompt_logits(oracle, p2))
    close(got[1], oracle_prompt_logits(oracle, p1))


def test_rows_of_a_slot_in_two_runs(paged, oracle):
    """A slot's rows split by another's: both runs see all earlier positions."""
    p = np.random.default_rng(5).integers(0, VOCAB, 12).tolist()
    o = np.random.default_rng(6).integers(0, VOCAB, 3).tolist()
    got = paged.forward(p[:5] + o + p[5:], list(range(5)) + list(range(3)) + list(range(5, 12)),
                        [1] * 5 + [2] * 3 + [1] * 7, [14, 7])
    close(got[0], oracle_prompt_logits(oracle, p))
    close(got[1], oracle_prompt_logits(oracle, o))


def test_pages_are_taken_and_returned(native, q8_model_bytes):
    h = native.Q8BatchHandle(0, q8_model_bytes, max_rows=64, slots=2, kv_type="bf16", page_size=8, pages=5)
    try:
        tok = list(range(100, 140))
        assert h.free_pages() == 5
        h.forward(tok[:9], range(9), [0] * 9)
        assert h.free_pages() == 3
        h.forward(tok[9:16], range(9, 16), [0] * 7)
        assert h.free_pages() == 3
        h.forward(tok[:24], range(24), [1] * 24)
        assert h.free_pages() == 0
        with pytest.raises(RuntimeError):
            h.forward(tok[16:17], [16], [0])
        h.release(1)
        assert h.free_pages() == 3
        h.forward(tok[16:17], [16], [0])
        assert h.free_pages() == 2
        h.forward(tok[:1], [0], [0])  # position 0 starts the slot anew
        assert h.free_pages() == 4
        with pytest.raises(RuntimeError):
            h.release(2)
    finally:
        h.close()


def test_a_call_without_pages_changes_nothing(native, q8_model_bytes, oracle):
    """Three slots start anew, but there are pages for two: the call fails, and all go on as they were."""
    p = np.random.default_rng(9).integers(0, VOCAB, 12).tolist()
    h = native.Q8BatchHandle(0, q8_model_bytes, max_rows=64, slots=3, kv_type="f32", page_size=8, pages=5)
    try:
        h.forward(p[:11], range(11), [0] * 11)
        assert h.free_pages() == 3
        with pytest.raises(RuntimeError):
            h.forward(p[:9] * 3, list(range(9)) * 3, [0] * 9 + [1] * 9 + [2] * 9)
        assert h.free_pages() == 3
        close(h.forward(p[11:], [11], [0], [0])[0], oracle_prompt_logits(oracle, p))
        h.forward(p[:9] * 2, list(range(9)) * 2, [0] * 9 + [1] * 9)
        assert h.free_pages() == 1
    finally:
        h.close()


@pytest.mark.parametrize("page_size,pages", [(16, None), (24, 4), (8, 10)])
def test_streams_through_few_pages(native, q8_model_bytes, oracle, page_size, pages):
    """Seven sequences with budgets 3..12 through three slots and a pool that holds them all,
    or about two: those without pages wait, and every stream is the oracle's."""
    h = native.Q8BatchHandle(0, q8_model_bytes, max_rows=128, slots=3, kv_type="f32", page_size=page_size, pages=pages)
    try:
        prompts = np.random.default_rng(21).integers(0, VOCAB, (7, 20))
        budgets = [3, 12, 5, 9, 4, 7, 12]
        toks, timing = h.generate_each(prompts, budgets)
        for i in range(7):
            ref, _ = oracle.generate(prompts[i].tolist(), budgets[i])
            assert toks[i] == ref, i
        assert timing.generated == sum(map(len, toks))
        total = h.free_pages()
        again, _ = h.generate_each(prompts, budgets, temperature=0.7, top_k=40, top_p=0.9, penalty=1.12, seed_base=5)
        assert h.free_pages() == total and len(again) == 7
    finally:
        h.close()


def test_a_sequence_larger_than_the_pool_fails(native, q8_model_bytes):
    h = native.Q8BatchHandle(0, q8_model_bytes, max_rows=128, slots=2, kv_type="f16", page_size=16, pages=2)
    try:
        prompts = np.random.default_rng(22).integers(0, VOCAB, (2, 30))
        with pytest.raises(RuntimeError):
            h.generate(prompts, 8)
        toks, _ = h.generate(prompts, 2)
        assert [len(t) for t in toks] == [2, 2]
    finally:
        h.close()


@pytest.mark.parametrize("kv_type,u", [("f16", 2.0 ** -11), ("bf16", 2.0 ** -8)])
def test_16_bit_pages(native, q8_model_bytes, oracle, kv_type, u):
    """Queries, keys, values, weights and outputs are rounded once per layer, each by u at
    most: five roundings of an attention output's inputs in each of 24 layers move the logits
    by no more than 5 * 24 * u / sqrt(3) of their norm if they only add up (a rounding's root
    mean square is at most u / sqrt(3))."""
    h = native.Q8BatchHandle(0, q8_model_bytes, max_rows=256, slots=2, kv_type=kv_type, page_size=32)
    try:
        prompt = np.random.default_rng(31).integers(0, VOCAB, 150).tolist()
        ref = oracle_prompt_logits(oracle, prompt)
        bound = 5 * 24 * u / 3 ** 0.5 * np.linalg.norm(ref)
        one = h.prefill(0, prompt)
        h.forward(prompt[:77], range(77), [1] * 77)
        h.forward(prompt[77:149], range(77, 149), [1] * 72)
        two = h.forward(prompt[149:], [149], [1], [0])[0]
        for got in (one, two):
            assert np.all(np.isfinite(got)) and np.linalg.norm(got - ref) <= bound
    finally:
        h.close()


def test_bench_prefill_and_launches(paged):
    assert paged.bench_prefill(256, 3, 1, 2) > 0
    assert paged.launches_per_step() == 2 + 24 * 12 + 3
