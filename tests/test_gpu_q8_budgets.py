"""The batched grouped-Q8 engine over several generate calls of one handle whose budgets
grow, so that its token buffer is made anew while a captured step exists."""
import numpy as np
import pytest

from test_gpu_q8_batch import VOCAB

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def oracle(oracle_lib, q8_model_bytes):
    return oracle_lib.Q8Oracle(q8_model_bytes)


@pytest.mark.parametrize("kv_type", [None, "f32"])
def test_budgets_that_grow(native, q8_model_bytes, oracle, kv_type):
    h = native.Q8BatchHandle(0, q8_model_bytes, max_rows=64, slots=2, kv_type=kv_type)
    try:
        prompts = np.random.default_rng(41).integers(0, VOCAB, (2, 9))
        for n_new in (2, 11, 5, 17):
            toks, _ = h.generate(prompts, n_new)
            for i in range(2):
                ref, _ = oracle.generate(prompts[i].tolist(), n_new)
                assert toks[i] == ref, (n_new, i)
    finally:
        h.close()
