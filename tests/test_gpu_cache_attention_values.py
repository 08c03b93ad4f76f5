"""CacheAttention of values and queries as large as their types have them, and of weights that are tiny."""
import math

import pytest
import torch

from _attention import FORMS
from qwen38_flash_ops_b200 import CacheAttention
from test_gpu_cache_attention import a_case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,group,tokens", [(64, 4, 1), (128, 8, 2), (256, 2, 1)])
@pytest.mark.parametrize("power", [40, 76, 90, 106, 112])
@pytest.mark.parametrize("some", [1, 7, 64])
def test_large_values(cuda, some, power, dim, group, tokens):
    """In eight bits, scales of every one, seventh or 64th token up to 2^107: values up to 2^115."""
    cache, table, q, n = a_case("e4m3", dim, 1, group, tokens, [300, 2000, 1], torch.bfloat16)
    flat = cache.v_scale.view(-1)
    flat[::some] = (flat[::some] * 2.0 ** power).clamp(max=2.0 ** 107)
    got, lse = CacheAttention()(q, cache, table, n, lse=True)
    check(got, lse, cache, table, q, n, 1 / math.sqrt(dim))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("power", [112, 122, 125])
def test_large_queries(cuda, form, power):
    """Queries up to BF16's largest exponent, with a scale that makes ordinary scores of them."""
    cache, table, q, n = a_case(form, 128, 2, 4, 2, [300, 65], torch.bfloat16)
    q[0] *= 2.0 ** power
    assert torch.isfinite(q).all()
    got, lse = CacheAttention(scale=2.0 ** -power)(q, cache, table, n, lse=True)
    check(got, lse, cache, table, q, n, 2.0 ** -power)
