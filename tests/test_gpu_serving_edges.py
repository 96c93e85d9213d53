"""Edges of the 8-bit attention: value scales far apart, NaN behind vanishing weights, rows that no sequence has, calls that repeat."""
import math

import numpy as np
import pytest
import torch

from oracle import serving_oracle as S
from test_gpu_serving_ops import DEV, EPS, _check_attention, _filled, _state, clean_status, gen, i32  # noqa: F401  (an autouse fixture)
from turboquant.kernels import _native
from turboquant.kernels.paged_8bit import allocate_cache_8bit, codes_and_scales, paged_attention_8bit

pytestmark = pytest.mark.gpu


# ---- denominators --------------------------------------------------------------------------------------
def _one_token_and_many(far, key, N, dtype, n, H, seqs, width, value=1.0):
    """Token 0 with score 0 and value scale `value`; N tokens with score `key` in pages whose value scale is 2^far smaller.  All sequences and heads are alike."""
    D, bs = 64, 16
    cache = allocate_cache_8bit(9, bs, H, DEV, D)
    codes, scales = codes_and_scales(cache, bs, D)
    g = gen(N)
    codes[:, :, :, 1] = (torch.randn(9, 1, 1, 16, D, generator=g, device=DEV) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    codes[1:, :, :, 0, :, 0] = torch.tensor(float(key), device=DEV).to(torch.float8_e4m3fn)
    codes[0, :, :, 0, 1:, 0] = torch.tensor(-448.0, device=DEV).to(torch.float8_e4m3fn)      # the other tokens of its page: weight e^-448
    scales[..., 0], scales[0, ..., 1], scales[1:, ..., 1] = 1.0, value, value * 2.0 ** -far
    L = 16 + N
    table = torch.cat([torch.zeros(1, dtype=torch.int32), 1 + torch.arange(N // 16, dtype=torch.int32) % 8])
    tables = torch.nn.functional.pad(table, (0, max(0, width - len(table)))).to(DEV).expand(seqs, -1).contiguous()
    q = torch.zeros(seqs * n, H, D, device=DEV, dtype=dtype)
    q[..., 0] = 1.0
    more = {} if n == 1 else dict(query_start_loc=torch.arange(seqs + 1, **i32) * n, max_query_len=n)
    got = paged_attention_8bit(q, cache, tables, torch.full((seqs,), L, **i32), bs, sm_scale=1.0, **more)
    c, s = _state(cache, bs, D)
    got = got.double().cpu().numpy().reshape(seqs, n, H, D)
    for j in {0, n - 1}:                                                    # the rows between see the same but for a few tokens
        want, tol = S.attention(q[:1, :1].double().cpu().numpy(), c[:, :1], s[:, :1], tables[:1].cpu().numpy(), [L - n + 1 + j], [0, 1], bs, 1.0, EPS[dtype])
        off = np.abs(got[:, j] - want) / tol
        assert off.max() <= 1, (off.max(), np.abs(got[0, j] / want - 1).max())


# clusters, the persistent kernel, prompt chunks whose keys one CTA walks over
_KERNELS = pytest.mark.parametrize("n,H,seqs,width", [(1, 8, 20, 0), (1, 8, 20, 9000), (1, 2, 1, 0), (40, 8, 10, 0)])


@_KERNELS
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("far,key,N", [(16, -11, 2048), (16, -11, 8192), (14, -12, 8192), (12, -14, 65536), (8, -16, 131072), (3, -20, 131072), (1, -20, 131072), (0, -20, 131072),
                                       (40, -10, 4096), (70, -3, 512)])
def test_denominators_keep_small_weights_of_small_values(far, key, N, dtype, n, H, seqs, width):
    """Many tokens of a weight that fp16 does not hold next to values 2^far larger count for the denominator."""
    _one_token_and_many(far, key, N, dtype, n, H, seqs, width)


@_KERNELS
@pytest.mark.parametrize("far,value,key", [(140, 2.0 ** 40, 0), (140, 2.0 ** 40, -5), (105, 2.0 ** 5, -20), (120, 2.0 ** 20, -10)])
def test_denominators_of_value_scales_as_far_apart_as_they_get(far, value, key, n, H, seqs, width):
    """Pages of zeros have the least scale, 2^-100: their weights count whatever the scale of the others is."""
    _one_token_and_many(far, key, 1024, torch.bfloat16, n, H, seqs, width, value)
