"""Edges of the 8-bit attention: value scales far apart, NaN behind vanishing weights, rows that no sequence has, calls that repeat."""
import math

import numpy as np
import pytest
import torch

from oracle import serving_oracle as S
from test_gpu_serving_ops import DEV, EPS, _check_attention, _filled, _state, clean_status, gen, i32  # noqa: F401  (an autouse fixture)
from turboquant.kernels import _native
from turboquant.kernels.block_plan import plan_step, release_blocks
from turboquant.kernels.paged_8bit import allocate_cache_8bit, codes_and_scales, paged_attention_8bit

pytestmark = pytest.mark.gpu


# ---- denominators --------------------------------------------------------------------------------------
def _one_token_and_many(far, key, N, dtype, n, H, seqs, width, value=1.0, lone=False):
    """Token 0 with score 0 and value scale `value`; N tokens with score `key` in pages whose value scale is 2^far smaller.  All sequences and heads are alike.
    lone: token 0 has values in four dims only."""
    D, bs = 64, 16
    cache = allocate_cache_8bit(9, bs, H, DEV, D)
    codes, scales = codes_and_scales(cache, bs, D)
    g = gen(N)
    codes[:, :, :, 1] = (torch.randn(9, 1, 1, 16, D, generator=g, device=DEV) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    if lone:
        codes.view(torch.uint8)[0, :, :, 1, :, 4:] = 0
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


@_KERNELS
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("far,key,N,value", [(16, -11, 2048, 64.0), (16, -11, 8192, 64.0), (14, -12, 8192, 64.0), (12, -14, 65536, 16.0), (8, -16, 131072, 4.0),
                                             (3, -20, 131072, 1.0), (2, -20, 131072, 1.0), (10, -3, 704, 16.0), (20, -9, 4096, 64.0), (22, -6, 1024, 128.0)])
def test_small_values_beside_zeros_of_a_page_of_large_ones(far, key, N, value, dtype, n, H, seqs, width):
    """In dims in which the large page holds zeros the output is made of the small values alone, at weights that are tiny next to its."""
    _one_token_and_many(far, key, N, dtype, n, H, seqs, width, value, lone=True)


@pytest.mark.parametrize("n,width", [(1, 0), (1, 40000), (4, 40000), (40, 0)])
@pytest.mark.parametrize("steps", [(0, -14, 3, -20, 0, -6, 5, -9), (5, 0, -6, -12, -17, 2, -8, -15), (-16, 0, -15, 1, -14, 2, -13, 3)])
def test_value_scales_that_rise_and_fall(steps, n, width):
    """Pages whose value scales go up and down by many powers of two, with values in dims of their own beside common ones: every page's dims are right."""
    g = gen(len(steps) + n)
    D, bs, H, L = 64, 16, 2, 1536
    cache, tables = _filled(g, [L], H, D, bs, spread=0)
    codes, scales = codes_and_scales(cache, bs, D)
    raw = codes.view(torch.uint8)
    for page in range(L // bs):
        k, b = page % len(steps), int(tables[0, page])
        scales[b, :, 0, 1] = 2.0 ** (steps[k] - 4)
        raw[b, :, 0, 1, :, 8:] &= 0x80
        raw[b, :, 0, 1, :, 8 + 7 * k:15 + 7 * k] |= torch.randint(0x30, 0x78, (H, 16, 7), generator=g, device=DEV, dtype=torch.uint8)
    tables = torch.nn.functional.pad(tables, (0, width), value=-9)
    q = (torch.randn(n, 4 * H, D, generator=g, device=DEV) * 2).half()
    more = {} if n == 1 else dict(query_start_loc=torch.tensor([0, n], **i32), max_query_len=n)
    got = paged_attention_8bit(q, cache, tables, torch.tensor([L], **i32), bs, **more)
    c, s = _state(cache, bs, D)
    want, tol = S.attention(q.double().cpu().numpy(), c, s, tables.cpu().numpy(), [L], [0, n], bs, D ** -0.5, EPS[torch.float16])
    off = np.abs(got.double().cpu().numpy() - want) / tol
    assert off.max() <= 1, off.max((0, 1))


# ---- NaN -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,width", [(1, 0), (1, 20000), (4, 0), (4, 20000), (40, 0)])
def test_nan_behind_a_vanishing_weight_reaches_the_output(n, width):
    """Values that are NaN in tokens whose scores lie 160 nats below the largest one: zero times NaN is NaN, wherever the work is cut."""
    D, bs, H, L = 128, 16, 2, 3000
    cache = allocate_cache_8bit(L // bs + 1, bs, H, DEV, D)
    codes, scales = codes_and_scales(cache, bs, D)
    raw = codes.view(torch.uint8)
    raw[:, :, :, 1] = torch.randint(0, 0x70, raw[:, :, :, 1].shape, generator=gen(3), device=DEV, dtype=torch.uint8)
    scales.fill_(1.0)
    codes[:, :, :, 0, :, 0] = torch.tensor(-160.0, device=DEV).to(torch.float8_e4m3fn)
    raw[0, :, 0, 0, 3, 0] = 0                                               # token 3 takes all
    dims = []
    for page in (1, 3, 15, 20, 47, 100, 180):                               # one dim for each page: of the same warp, CTA, a following and a far one
        raw[page, :, 0, 1, 7, page % D] = 0x7f
        dims.append(page % D)
    table = torch.arange(L // bs + 1, **i32)
    tables = torch.nn.functional.pad(table, (0, max(0, width - len(table))))[None]
    q = torch.zeros(n, 4 * H, D, device=DEV, dtype=torch.float16)
    q[..., 0] = 1.0
    more = {} if n == 1 else dict(query_start_loc=torch.tensor([0, n], **i32), max_query_len=n)
    got = paged_attention_8bit(q, cache, tables, torch.tensor([L], **i32), bs, sm_scale=1.0, **more)
    want = codes[0, :, 0, 1, 3].float().repeat_interleave(4, 0)
    want[:, dims] = math.nan
    assert torch.equal(got.isnan(), want.isnan().expand(n, -1, -1))
    fine = ~want.isnan().expand(n, -1, -1)
    assert torch.equal(got[fine], want.half().expand(n, -1, -1)[fine])


@pytest.mark.parametrize("width", [0, 20000])
@pytest.mark.parametrize("n,G", [(4, 2), (8, 1), (5, 4), (8, 4)])
def test_nan_of_a_few_queries_reaches_what_sees_it_and_nothing_else(n, G, width):
    """A NaN value that the later queries see and the earlier ones do not, and a NaN key, in the kernels for up to 32 rows."""
    g = gen(n * G)
    cache, tables = _filled(g, [60, 60], 1, 128, 16)
    codes, _ = codes_and_scales(cache, 16)
    raw = codes.view(torch.uint8)
    t = 60 - n + 2                                                          # seen from query 2 on
    raw[int(tables[0, t // 16]), 0, 0, 1, t % 16, 77] = 0xff
    raw[int(tables[1, t // 16]), 0, 0, 0, t % 16, 3] = 0x7f
    tables = torch.nn.functional.pad(tables, (0, width), value=-9)
    q = torch.randn(2 * n, G, 128, generator=g, device=DEV).half()
    starts, lens = torch.tensor([0, n, 2 * n], **i32), torch.tensor([60, 60], **i32)
    got = paged_attention_8bit(q, cache, tables, lens, 16, query_start_loc=starts, max_query_len=n)
    c, s = _state(cache, 16, 128)
    want, tol = S.attention(q.double().cpu().numpy(), c, s, tables.cpu().numpy(), [60, 60], [0, n, 2 * n], 16, 128 ** -0.5, EPS[torch.float16])
    g64 = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(g64), np.isnan(want))
    assert np.isnan(g64[2:n, :, 77]).all() and not np.isnan(g64[:2]).any() and np.isnan(g64[n + 2:]).all()
    fine = ~np.isnan(want)
    assert (np.abs(g64 - want)[fine] <= tol[fine]).all()


# ---- rows that no sequence has -----------------------------------------------------------------------------
def _after_garbage(q, *args, **kw):
    """The call, with the allocator's block for its result full of NaN."""
    junk = [torch.full_like(q, math.nan) for _ in range(3)]
    del junk
    return paged_attention_8bit(q, *args, **kw)


@pytest.mark.parametrize("queries,lens,G,most,width", [
    ([2, 3, 5], [20, 30, 40], 2, 3, 0), ([2, 3, 5], [20, 30, 40], 2, 3, 9000), ([2, 9, 0, 10], [20, 30, 7, 40], 4, 8, 0),
    ([2, 9, 0, 10], [20, 30, 7, 40], 4, 8, 9000), ([70, 1, 90], [70, 5, 300], 4, 66, 0), ([70, 1, 0, 90, 3], [70, 5, 4, 300, 30], 4, 66, 9000)])
def test_rows_that_are_left_out_or_that_no_sequence_has_are_zeros(queries, lens, G, most, width):
    """Rows before the first sequence, behind the last one and beyond max_query_len: zeros in a new result, left as they were in `out`."""
    g = gen(sum(queries))
    cache, tables = _filled(g, lens, 2, 128, 16)
    tables = torch.nn.functional.pad(tables, (0, width), value=-9)
    ahead, behind, T = 3, 4, sum(queries)
    q = torch.randn(ahead + T + behind, 2 * G, 128, generator=g, device=DEV).half()
    lens_t = torch.tensor(lens, **i32)
    starts = torch.tensor(np.concatenate([[0], np.cumsum(queries)]) + ahead, **i32)
    got = _after_garbage(q, cache, tables, lens_t, 16, query_start_loc=starts, max_query_len=most)
    assert _native.read_status(DEV) == _native.STATUS_TOO_LONG
    out = torch.full_like(q, 7.0)
    paged_attention_8bit(q, cache, tables, lens_t, 16, query_start_loc=starts, max_query_len=most, out=out)
    assert _native.read_status(DEV) == _native.STATUS_TOO_LONG
    c, s = _state(cache, 16, 128)
    # a sequence that is cut is served as if its first rows were all of them
    cut = [min(n, most) for n in queries]
    served = torch.zeros(len(q), dtype=torch.bool, device=DEV)
    for i, n in enumerate(cut):
        a = int(starts[i])
        served[a:a + n] = True
        want, tol = S.attention(q[a:a + n].double().cpu().numpy(), c, s, tables[i:i + 1].cpu().numpy(), [lens[i]], [0, n], 16, 128 ** -0.5, EPS[torch.float16])
        assert (np.abs(got[a:a + n].double().cpu().numpy() - want) <= tol).all()
    assert not got[~served].any() and (out[~served] == 7).all() and torch.equal(got[served], out[served])


def test_offsets_that_are_none_touch_nothing_else():
    g = gen(17)
    cache, tables = _filled(g, [64, 64, 64], 2, 128, 16)
    q = torch.randn(3, 4, 128, generator=g, device=DEV).bfloat16()
    wild = torch.tensor([2, -7, 1 << 30, 3], **i32)                         # sequence 1 is cut to the tensor's rows, the others have none
    around = torch.full((9, 4, 128), 7.0, device=DEV, dtype=torch.bfloat16)
    paged_attention_8bit(q, cache, tables, torch.tensor([64, 64, 64], **i32), 16, query_start_loc=wild, max_query_len=2, out=around[3:6])
    assert _native.read_status(DEV) == _native.STATUS_TOO_LONG
    assert (around[:3] == 7).all() and (around[5:] == 7).all() and torch.isfinite(around).all()


# ---- scales and sizes in the kernel for prompt chunks ------------------------------------------------------
def test_prompt_chunks_with_negative_and_zero_scales():
    for dtype in (torch.float16, torch.bfloat16):
        _check_attention(gen(5), [300, 40], [40, 40], 8, 2, 128, 16, dtype, sm_scale=-0.05)
        _check_attention(gen(6), [300, 40], [40, 40], 8, 2, 128, 16, dtype, sm_scale=0.0)


def test_prompt_chunks_with_scores_of_any_size():
    _check_attention(gen(1), [300, 40], [40, 40], 8, 2, 128, 16, torch.float16, q_size=30.0, spread=0, sm_scale=0.02)
    _check_attention(gen(2), [300, 40], [40, 40], 8, 2, 128, 16, torch.bfloat16, spread=40, sm_scale=2.0 ** -45)
    _check_attention(gen(3), [300, 40], [40, 40], 8, 2, 128, 16, torch.bfloat16, q_size=1e30, sm_scale=1e-32)
    _check_attention(gen(4), [300, 40], [40, 40], 8, 2, 128, 16, torch.bfloat16, q_size=1e-30, sm_scale=1e28)


# ---- repetition --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("queries,lens,width", [([1], [5000], 0), ([1] * 40, [700] * 40, 0), ([1] * 30, [100 * i + 1 for i in range(30)], 9000),
                                                ([300, 200], [3000, 900], 0), ([1, 1, 300, 2, 1], [900, 70, 1200, 33, 400], 9000)])
def test_repeated_calls_are_equal_bit_for_bit(queries, lens, width):
    g = gen(len(queries))
    cache, tables = _filled(g, lens, 2, 128, 16)
    tables = torch.nn.functional.pad(tables, (0, width), value=-9)
    q = torch.randn(sum(queries), 16, 128, generator=g, device=DEV).half()
    starts = torch.tensor(np.concatenate([[0], np.cumsum(queries)]), **i32)
    call = lambda: paged_attention_8bit(q, cache, tables, torch.tensor(lens, **i32), 16, query_start_loc=starts, max_query_len=max(queries))
    first = call()
    for _ in range(20):
        assert torch.equal(call(), first)


# ---- calls that nothing above makes ----------------------------------------------------------------------------
@pytest.mark.parametrize("Hq,H,n,width", [(33, 1, 5, 0), (71, 1, 5, 0), (128, 1, 3, 9000), (257, 1, 3, 0), (80, 2, 140, 0), (40, 1, 900, 0)])
def test_single_queries_of_large_groups(Hq, H, n, width):
    """More than 32 query heads on a KV head: single tokens in the kernel for prompt chunks, without offsets, up to more sequences than are ranked."""
    lens = [(37 * i) % 200 for i in range(n - 1)] + [700]
    _check_attention(gen(Hq), lens, [1] * n, Hq, H, 64, 16, torch.bfloat16 if n > 10 else torch.float16, width=width)


@pytest.mark.parametrize("n,width", [(1, 0), (1, 20000), (3, 0), (3, 20000), (30, 0)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_query_that_is_no_number_spoils_its_own_row_only(n, width, dtype):
    g = gen(n)
    cache, tables = _filled(g, [300, 90], 2, 128, 16)
    tables = torch.nn.functional.pad(tables, (0, width), value=-9)
    q = torch.randn(2 * n, 8, 128, generator=g, device=DEV).to(dtype)
    more = {} if n == 1 else dict(query_start_loc=torch.tensor([0, n, 2 * n], **i32), max_query_len=n)
    lens = torch.tensor([300, 90], **i32)
    clean = paged_attention_8bit(q, cache, tables, lens, 16, **more)
    q[0, 3, 17], q[2 * n - 1, 5, 100] = math.nan, math.inf
    got = paged_attention_8bit(q, cache, tables, lens, 16, **more)
    spoilt = torch.zeros(2 * n, 8, dtype=torch.bool, device=DEV)
    spoilt[0, 3] = spoilt[2 * n - 1, 5] = True
    assert got[spoilt].isnan().all() and torch.equal(got[~spoilt], clean[~spoilt])


@pytest.mark.parametrize("queries,lens,width", [([1] * 9, [900] * 9, 0), ([1] * 20, [100 * i + 1 for i in range(20)], 9000), ([90, 40], [3000, 100], 0),
                                                ([1, 1, 200, 2], [900, 70, 700, 33], 9000)])
def test_the_result_may_take_the_queries_place(queries, lens, width):
    g = gen(len(queries))
    cache, tables = _filled(g, lens, 2, 64, 16)
    tables = torch.nn.functional.pad(tables, (0, width), value=-9)
    q = torch.randn(sum(queries), 12, 64, generator=g, device=DEV).half()
    call = dict(query_start_loc=torch.tensor(np.concatenate([[0], np.cumsum(queries)]), **i32), max_query_len=max(queries))
    want = paged_attention_8bit(q, cache, tables, torch.tensor(lens, **i32), 16, **call)
    assert paged_attention_8bit(q, cache, tables, torch.tensor(lens, **i32), 16, out=q, **call) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("queries,lens,width", [([1] * 30, [100 * i + 1 for i in range(30)], 9000), ([300, 200], [3000, 900], 0), ([1, 1, 300, 2], [900, 70, 1200, 33], 9000)])
def test_two_calls_at_once(queries, lens, width):
    """Calls on two streams, each with a workspace of its own: those of one do not show in the other's."""
    problems = []
    for seed in (1, 2):
        g = gen(seed)
        cache, tables = _filled(g, lens, 2, 128, 16)
        tables = torch.nn.functional.pad(tables, (0, width), value=-9)
        q = torch.randn(sum(queries), 16, 128, generator=g, device=DEV).half()
        starts = torch.tensor(np.concatenate([[0], np.cumsum(queries)]), **i32)
        args, kw = (q, cache, tables, torch.tensor(lens, **i32), 16), dict(query_start_loc=starts, max_query_len=max(queries))
        problems.append((args, kw, paged_attention_8bit(*args, **kw)))
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(15):
        for stream, (args, kw, _), out in zip(streams, problems, outs):
            with torch.cuda.stream(stream):
                out.append(paged_attention_8bit(*args, **kw))
    torch.cuda.synchronize()
    for (_, _, want), out in zip(problems, outs):
        assert all(torch.equal(o, want) for o in out)


# ---- numbers beyond 32 bits --------------------------------------------------------------------------------
@pytest.mark.parametrize("most", [100, (1 << 27) + 5, (1 << 31) - 1, (1 << 32) + 1, 1 << 40])
def test_any_bound_of_the_queries_will_do(most):
    """max_query_len only has to be large enough."""
    g = gen(8)
    cache, tables = _filled(g, [40, 300, 9], 2, 64, 16)
    q = torch.randn(6, 64, 64, generator=g, device=DEV).half()
    starts, lens = torch.tensor([0, 1, 4, 6], **i32), torch.tensor([40, 300, 9], **i32)
    want = paged_attention_8bit(q, cache, tables, lens, 16, query_start_loc=starts, max_query_len=3)
    c, s = _state(cache, 16, 64)
    ref, tol = S.attention(q.double().cpu().numpy(), c, s, tables.cpu().numpy(), [40, 300, 9], [0, 1, 4, 6], 16, 0.125, EPS[torch.float16])
    assert (np.abs(want.double().cpu().numpy() - ref) <= tol).all()
    for out in (None, torch.full_like(q, 7.0)):
        got = paged_attention_8bit(q, cache, tables, lens, 16, query_start_loc=starts, max_query_len=most, out=out)
        assert (np.abs(got.double().cpu().numpy() - ref) <= tol).all() and (out is None or got is out)


def test_block_sizes_beyond_32_bits_are_refused():
    v, t, c = torch.ones(2, **i32), torch.zeros(2, 4, **i32), torch.ones(1, **i32)
    with pytest.raises(ValueError, match="block_size"):
        plan_step(v, v, t, v, c, (1 << 32) + 16, 2)
    with pytest.raises(ValueError, match="block_size"):
        release_blocks(v.bool(), v, t, v, c, (1 << 32) + 16)
