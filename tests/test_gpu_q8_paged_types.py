"""The batched grouped-Q8 engine on fp16 and bf16 pages against the oracle, whose cache is fp32.

Five roundings a layer reach its output: queries, keys, values, attention weights and attention
outputs, each by u at most and by u / sqrt(3) in root mean square.  They are independent, so that
over 24 layers they add up as squares: sqrt(5 * 24) u / sqrt(3) of the logits' norm, were the
attention all that a layer adds to its input."""
import numpy as np
import pytest

from test_gpu_q8_batch import VOCAB, oracle_prompt_logits

pytestmark = pytest.mark.gpu
UNITS = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def oracle(oracle_lib, q8_model_bytes):
    return oracle_lib.Q8Oracle(q8_model_bytes)


def share(kv_type):
    return (5 * 24 / 3) ** 0.5 * UNITS[kv_type]


@pytest.mark.parametrize("kv_type", ["f16", "bf16"])
@pytest.mark.parametrize("page_size,n", [(8, 33), (32, 150), (64, 200)])
def test_logits(native, q8_model_bytes, oracle, kv_type, page_size, n):
    """A prompt in one piece, in two with a single token behind them, and token by token."""
    h = native.Q8BatchHandle(0, q8_model_bytes, max_rows=256, slots=3, kv_type=kv_type, page_size=page_size)
    try:
        prompt = np.random.default_rng(n).integers(0, VOCAB, n).tolist()
        ref = oracle_prompt_logits(oracle, prompt)
        got = [h.prefill(0, prompt)]
        h.forward(prompt[:n // 2], range(n // 2), [1] * (n // 2))
        h.forward(prompt[n // 2:-1], range(n // 2, n - 1), [1] * (n - 1 - n // 2))
        got.append(h.forward(prompt[-1:], [n - 1], [1], [0])[0])
        if n < 100:
            for i, t in enumerate(prompt):
                one = h.forward([t], [i], [2], [0])[0]
            got.append(one)
        for x in got:
            print(kv_type, n, np.linalg.norm(x - ref) / np.linalg.norm(ref), share(kv_type))
            assert np.linalg.norm(x - ref) <= share(kv_type) * np.linalg.norm(ref)
    finally:
        h.close()


@pytest.mark.parametrize("kv_type", ["f16", "bf16"])
def test_tokens(native, q8_model_bytes, oracle, kv_type):
    """Every token of a greedy stream is, given those before it, the oracle's own or one whose logit is
    below the oracle's best by no more than both can be off: six times the logits' root mean square
    of that share, each."""
    h = native.Q8BatchHandle(0, q8_model_bytes, max_rows=64, slots=2, kv_type=kv_type, page_size=16, pages=9)
    try:
        prompts = np.random.default_rng(51).integers(0, VOCAB, (4, 20))
        toks, _ = h.generate_each(prompts, [14, 5, 9, 14])
        same = 0
        for p, stream in zip(prompts, toks):
            oracle.reset()
            seq = p.tolist() + stream
            for i, t in enumerate(seq[:-1]):
                ref = oracle.forward(t, i, i >= 19)
                if i >= 19:
                    best = float(np.max(ref[:151643]))
                    assert best - ref[seq[i + 1]] <= 12 * share(kv_type) * np.linalg.norm(ref) / VOCAB ** 0.5
                    same += best == ref[seq[i + 1]]
        print(kv_type, "the oracle's own:", same, "of", sum(map(len, toks)))
        assert same >= sum(map(len, toks)) / 2
    finally:
        h.close()
