"""That the check of chunks sees a chunk which is missing or counted twice: results made on the CPU, with and without such a mistake."""
import numpy as np
import pytest
import torch

from tests.test_gpu_cache4_parts import ONE, check_marks


def result(before, new, heads, kv_heads, dim, dtype, chunk=32, wrong=None, times=1):
    """What attention over marked values gives where the positions of one chunk count `times` times for head 0 of sequence 0."""
    rows = []
    for b, (a, n) in enumerate(zip(before, new)):
        for i in range(n):
            p = np.arange(a + i + 1)
            per_head = []
            for g in range(kv_heads):
                w = np.ones(len(p))
                if b == 0 and g == 0 and wrong is not None:
                    w[p // chunk == wrong] = times
                per_head += [np.bincount((p // chunk + g + 5 * b) % dim, w, dim) * ONE / w.sum()] * (heads // kv_heads)
            rows.append(per_head)
    return torch.from_numpy(np.array(rows)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("before,new,heads,kv_heads,dim", [([20000], [1], 4, 1, 64), ([300, 40], [3, 1], 4, 2, 64), ([131000], [1], 2, 1, 128), ([16000], [2], 2, 1, 128)])
def test_a_chunk_more_or_less_is_seen(dtype, before, new, heads, kv_heads, dim):
    case = (before, new, heads, kv_heads, dim)
    check_marks(result(*case, dtype), *case, 32, dtype)
    last = before[0] // 32 - 1
    for wrong in (0, last // 2, last):
        for times in (0, 2):
            with pytest.raises(AssertionError):
                check_marks(result(*case, dtype, wrong=wrong, times=times), *case, 32, dtype)
