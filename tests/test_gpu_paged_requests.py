"""More requests than a workgroup has threads, so that a thread counts the steps of several, in the chunk kernel (an average of more than 16
rows a request and kv head) and, for comparison, in the decode kernel."""
import random

import pytest
import torch

from test_gpu_paged import BF16, F16, Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,d,dtype,window,most", [(257, 64, F16, 0, 9), (700, 64, BF16, 50, 9), (300, 128, F16, 0, 12), (513, 128, BF16, 0, 9),
                                                          (513, 256, F16, 0, 9), (1100, 256, BF16, 33, 9), (600, 128, F16, 0, 1)])
def test_requests_beyond_the_threads(requests, d, dtype, window, most):
    rng = random.Random(requests)
    lens = [(rng.choice([0, rng.randrange(150)]), rng.randint(most // 2, most) if rng.random() < 0.9 else 0) for _ in range(requests)]
    lens[0] = lens[-1] = (0, 0)
    lens[requests // 2] = (900, 40)
    rows = 5 * sum(n for _, n in lens) / requests
    assert (rows > 16) == (most > 1)
    Batch(lens, 5, 1, d, dtype, seed=requests, pad=3).check(window=window)
    torch.cuda.empty_cache()
