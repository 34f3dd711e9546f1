"""The decoder's cache modes and branches where a call fails, or ends a range."""

import numpy as np
import pytest

from oracle.llama import make_llama
from test_gpu_text_cache import decoder, toks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv,width", [(4, 3, 256), (2, 4, 512)])
def test_heads_that_kv_heads_do_not_divide_are_refused(gpu, oracle, heads, kv, width):
    """The f32 cache maps any number of heads to the kv heads, the 8-bit cache
    whole groups only."""
    from eosllm_b200.text import TextDecoder
    d = decoder(make_llama(oracle, max_ctx=16, n_embd=width, n_head=heads, n_kv_head=kv), q8=False)
    with pytest.raises(gpu.CudaBackendError) as ex:
        d.set_cache(TextDecoder.CACHE_Q8)
    assert ex.value.status == gpu.EOS_E_UNSUPPORTED and "multiple of n_kv_head" in str(ex.value)
    d.close()


def test_a_cache_whose_step_cannot_be_recorded_changes_nothing(gpu, oracle):
    """The failure comes when the new cache is there and the step is recorded for
    it (three kv heads for four heads): the decoder keeps its cache, its step and
    its results, however often it is asked."""
    from eosllm_b200.text import TextDecoder
    model = make_llama(oracle, max_ctx=16, n_kv_head=3)
    d = decoder(model, q8=False)
    first, kernels = [d.step(t) for t in (3, 7)], d.step_kernels
    for _ in range(3):
        d.reset()
        with pytest.raises(gpu.CudaBackendError):
            d.set_cache(TextDecoder.CACHE_Q8)
        assert d.cache == TextDecoder.CACHE_F32 and d.step_kernels == kernels
        for t, w in zip((3, 7), first):
            assert np.array_equal(d.step(t), w)
    d.reset()
    d.set_cache(TextDecoder.CACHE_F32)  # the one it has
    assert np.array_equal(d.step(3), first[0])
    d.close()


@pytest.mark.parametrize("temperature", [1e-45, 1e-42, 2.9e-39, 1e-38, 1e-30])
def test_the_smallest_temperatures_draw_the_most_likely_token(gpu, oracle, temperature):
    """A positive temperature whose reciprocal no f32 holds is a temperature like
    the others: as it goes to 0 the largest logit takes all."""
    model = make_llama(oracle, max_ctx=64)
    d = decoder(model)
    d.prefill(toks(17, 320, 1))
    d.fork(2, 8)
    a = d.branch_step([[5], [9]], [[0.3], [0.999]], temperature=0.0)
    d.close_branches()
    d.fork(2, 8)
    b = d.branch_step([[5], [9]], [[0.3], [0.999]], temperature=temperature)
    assert [list(x) for x in a] == [list(x) for x in b]
    d.close()
