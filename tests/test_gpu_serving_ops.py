"""Rotary positions, the 8-bit paged cache with its attention, and step tables, against their definitions in 64 bits."""
import math

import numpy as np
import pytest
import torch

from oracle import serving_oracle as S
from turboquant.kernels import _native
from turboquant.kernels.block_plan import plan_step, release_blocks
from turboquant.kernels.paged_8bit import allocate_cache_8bit, codes_and_scales, paged_attention_8bit, quantize_and_scatter
from turboquant.kernels.rotary import make_rotary_table, rotary_embedding

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7, torch.float32: 2.0 ** -23}
i32 = dict(dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.fixture(autouse=True)
def clean_status():
    _native.read_status(DEV)
    yield
    assert _native.read_status(DEV) == 0, "a call raised a status bit that its test did not read"


# ---- rotary -------------------------------------------------------------------------------------------
def _check_rotary(got, x, table, pos, interleaved, inverse):
    half = table.shape[1] // 2
    t = table.double().cpu().numpy()[pos.cpu().numpy()]
    y, R = x.double().cpu().numpy().copy(), table.shape[1]
    c, s = t[:, None, :half], t[:, None, half:] * (-1 if inverse else 1)
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, half), slice(half, R))
    u, w = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    bound = np.zeros_like(y)
    bound[..., a], bound[..., b] = np.abs(u * c) + np.abs(w * s), np.abs(w * c) + np.abs(u * s)
    # half a step of the type, and two fp32 roundings of terms no larger than the sum of their sizes
    tol = np.abs(y) * EPS[x.dtype] / 2 + bound * 2.0 ** -23 + (2.0 ** -25 if x.dtype == torch.float16 else 0)
    g = got.double().cpu().numpy()
    assert (np.abs(g - y) <= tol).all(), np.abs(g - y).max()
    assert np.array_equal(g[..., R:], y[..., R:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,hq,hk,D,R", [(1, 1, 1, 64, 64), (3, 32, 8, 128, 128), (1025, 12, 4, 128, 64), (77, 5, 1, 80, 20), (40, 3, 2, 96, 24),
                                         (130, 8, 8, 256, 256), (9, 2, 1, 7, 6), (2000, 2, 1, 10, 2), (700, 64, 8, 128, 128)])
def test_rotary(T, hq, hk, D, R, dtype, interleaved):
    if interleaved and D % 2:
        D += 1
    g = gen(T)
    qkv = torch.randn(T, hq + 2 * hk, D, generator=g, device=DEV).to(dtype)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    table = make_rotary_table(R, 4096, device=DEV)
    pos = torch.randint(0, 4096, (T,), generator=g, device=DEV, dtype=torch.int64 if T % 2 else torch.int32)
    for inverse in (False, True):
        a, b = rotary_embedding(q, k, pos, table, interleaved=interleaved, inverse=inverse)
        _check_rotary(a, q, table, pos, interleaved, inverse)
        _check_rotary(b, k, table, pos, interleaved, inverse)
        assert a.is_contiguous() and b.is_contiguous()


def test_rotary_in_place_without_keys_and_of_no_rows():
    g = gen(1)
    table = make_rotary_table(64, 512, device=DEV)
    qkv = torch.randn(33, 12, 128, generator=g, device=DEV).half()
    before, pos = qkv.clone(), torch.arange(33, device=DEV)
    q, k = qkv[:, :8], qkv[:, 8:10]
    want = rotary_embedding(q, k, pos, table)
    res = rotary_embedding(q, k, pos, table, out=(q, k))
    assert res[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 10:], before[:, 10:])
    alone, none = rotary_embedding(before[:, :8], None, pos, table)
    assert none is None and torch.equal(alone, want[0])
    a, b = rotary_embedding(qkv[:0, :8], qkv[:0, 8:10], pos[:0], table)
    assert a.shape == (0, 8, 128) and b.shape == (0, 2, 128)
    a, b = rotary_embedding(qkv[:, :0], k, pos, table)
    assert a.shape == (33, 0, 128) and b.shape == (33, 2, 128)


def test_rotary_is_undone_by_its_inverse_and_is_its_gradient():
    """<turn(x), y> = <x, turn^-1(y)>: the gradient of a turn is the inverse turn, by the formula and by differences."""
    g = gen(2)
    table = make_rotary_table(96, 64, device=DEV)
    x, y = (torch.randn(20, 4, 128, generator=g, device=DEV) for _ in range(2))
    pos = torch.randint(0, 64, (20,), generator=g, device=DEV)
    turn = lambda t, inv=False: rotary_embedding(t, None, pos, table, inverse=inv)[0]
    torch.testing.assert_close(turn(turn(x), True), x, atol=4e-6, rtol=0)      # four roundings of values up to 5, 2^-24 each
    left, right = (turn(x).double() * y.double()).sum(), (x.double() * turn(y, True).double()).sum()
    assert abs(left - right) <= 20 * 4 * 128 * 16 * 2.0 ** -23
    d = torch.zeros_like(x)
    d[3, 2, 5] = 0.5                                                            # the turn is linear: a difference of any size is its slope
    slope = ((turn(x + d).double() - turn(x).double()) * y.double()).sum() / 0.5
    assert abs(slope - turn(y, True)[3, 2, 5].double()) <= 1e-5


def test_rotary_positions_outside_the_table_are_clamped_and_flagged():
    table = make_rotary_table(128, 16, device=DEV)
    q = torch.randn(3, 2, 128, generator=gen(3), device=DEV).bfloat16()
    got, _ = rotary_embedding(q, None, torch.tensor([-1, 16, 1 << 40], device=DEV), table)
    assert _native.read_status(DEV) == _native.STATUS_BAD_POSITION
    want, _ = rotary_embedding(q, None, torch.tensor([0, 15, 15], device=DEV), table)
    assert torch.equal(got, want)


def test_rotary_refusals():
    q, table, pos = torch.zeros(4, 2, 128, device=DEV, dtype=torch.float16), make_rotary_table(128, 16, device=DEV), torch.arange(4, device=DEV)
    bad = [dict(q=q[..., 0]), dict(q=q.double()), dict(k=q.bfloat16()), dict(k=q[:3]), dict(positions=pos[:3]), dict(cos_sin=table.half()),
           dict(cos_sin=table[:, :127].contiguous()), dict(cos_sin=make_rotary_table(256, 4, device=DEV)), dict(q=q.transpose(1, 2)),
           dict(positions=pos.float()), dict(cos_sin=table[:, ::2])]
    for change in bad:
        with pytest.raises(ValueError):
            rotary_embedding(**{**dict(q=q, k=q, positions=pos, cos_sin=table), **change})
    with pytest.raises(RuntimeError, match="no autograd"):
        rotary_embedding(q.requires_grad_(), None, pos, table, out=(q, None))


# ---- the 8-bit cache ---------------------------------------------------------------------------------------
def _state(cache, bs, D):
    codes, scales = codes_and_scales(cache, bs, D)
    return codes.view(torch.uint8).cpu().numpy().copy(), scales.double().cpu().numpy()


def _append_both(cache, key, value, slots, bs):
    """The call, and the oracle on the state before it; codes and scales have to be equal (but for the sign of a NaN)."""
    D = key.shape[-1]
    codes, scales = _state(cache, bs, D)
    quantize_and_scatter(key, value, cache, slots, bs)
    S.append(codes, scales, key.double().cpu().numpy(), value.double().cpu().numpy(), slots.tolist(), bs)
    got_codes, got_scales = _state(cache, bs, D)
    np.testing.assert_array_equal(got_scales, scales)
    np.testing.assert_array_equal(S.e4m3_decode(got_codes), S.e4m3_decode(codes))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,H,bs", [(128, 2, 16), (64, 3, 32), (128, 1, 48)])
def test_append_step_by_step(D, H, bs, dtype):
    """Prompts of ragged lengths, then single tokens and small groups that continue their pages, growing in size."""
    g = gen(D + H)
    cache = allocate_cache_8bit(12, bs, H, DEV, D)
    cache.random_(0, 256, generator=g)                                     # whatever a page held before it is begun does not matter ...
    codes_and_scales(cache, bs, D)[0].view(torch.uint8).bitwise_and_(0x77)     # (but codes that are left alone are compared as numbers)
    blocks = torch.randperm(12, generator=g, device=DEV).tolist()
    lens = [0, 0, 0]
    slot = lambda s, p: blocks[4 * s + p // bs] * bs + p % bs
    for step, new in enumerate([(33, 1, 16), (1, 1, 1), (1, 14, 1), (3, 1, 0), (1, 2, 15), (1, 1, 1)]):
        slots = [slot(s, lens[s] + j) for s in range(3) for j in range(new[s])]
        lens = [a + b for a, b in zip(lens, new)]
        x = torch.randn(2, len(slots), H, D, generator=g, device=DEV) * 2.0 ** (2 * step - 8)
        x[:, :, :, 5] *= 10
        _append_both(cache, *x.to(dtype), torch.tensor(slots, device=DEV), bs)


def test_append_scales_at_their_borders():
    """Largest values at 448 * 2^e and just above, zeros, the smallest and the largest numbers, infinities and NaN."""
    D, bs = 128, 16
    cache = allocate_cache_8bit(16, bs, 1, DEV)
    rows = torch.zeros(14, 1, D, device=DEV)
    for i, v in enumerate([448.0, 448.0 * (1 + 2.0 ** -23), 3.5, 3.5000002, 0.0, 1e-38, 2.0 ** -101 * 448, 3.4e38, math.inf, -math.inf, math.nan, 1.0,
                           2.0 ** -130, 1e-45]):
        rows[i, 0, :3] = torch.tensor([v, -v / 3, v / 1000])
    rows[8, 0, 4] = 2.0
    _append_both(cache, rows, rows.flip(0).contiguous(), torch.arange(14, device=DEV) * 16, bs)
    codes, scales = codes_and_scales(cache, bs)
    assert scales[0, 0, 0, 0] == 1 and scales[1, 0, 0, 0] == 2 and scales[4, 0, 0, 0] == 2.0 ** -100
    assert codes[8, 0, 0, 0, 0, 0].float() == 448 and codes[10, 0, 0, 0, 0, 0].float().isnan()
    # a page that holds an infinity and a NaN goes on
    _append_both(cache, torch.full((1, 1, D), 7.0, device=DEV), torch.full((1, 1, D), 1e30, device=DEV), torch.tensor([8 * 16 + 1], device=DEV), bs)


def test_append_many_rows_in_every_window():
    """Calls around the sizes at which the blocks' windows change, as single rows and as prompts, with skipped rows between."""
    D, bs, H = 64, 16, 2
    for T in (1, 2, 15, 17, 511, 513, 4095, 4097, 4500):
        g = gen(T)
        x = torch.randn(2, T, H, D, generator=g, device=DEV).half()
        single = torch.randperm(T, generator=g, device=DEV) * bs + torch.randint(0, bs, (T,), generator=g, device=DEV)
        single[::7] = -1
        prompt = torch.arange(T, device=DEV) + 5
        for slots in (single, prompt):
            cache = allocate_cache_8bit(T + 2, bs, H, DEV, D)
            quantize_and_scatter(*x, cache, slots, bs)
            codes, scales = codes_and_scales(cache, bs, D)
            keep = slots >= 0
            for kv in range(2):
                v = codes.view(torch.uint8)[slots[keep] // bs, :, 0, kv, slots[keep] % bs].view(torch.float8_e4m3fn).float()
                s = scales[slots[keep] // bs, :, 0, kv]
                v = v * s[..., None]
                want = x[kv][keep].float()
                # half a step of e4m3, or of its subnormals: 2^-4 relative, 2^-10 of the scale
                assert ((v - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, s[..., None] * 2.0 ** -10)).all()
                assert (s >= 2.0 ** -9).all() and (s <= 2.0 ** -6).all()
            touched = torch.zeros(T + 2, bs, dtype=torch.bool, device=DEV)
            touched.view(-1)[slots[keep]] = True
            rest = codes.view(torch.uint8)[:, :, 0].permute(0, 3, 1, 2, 4)[~touched]
            assert not rest.any()


def test_append_slots_that_are_skipped_and_views():
    D, bs, H = 128, 32, 2
    g = gen(5)
    cache = allocate_cache_8bit(3, bs, H, DEV)
    qkv = torch.randn(20, 8 * D, generator=g, device=DEV).bfloat16().view(20, 8, D)
    slots = torch.tensor([-1, -5, 0, 1, 2, 3 * bs, 1 << 40, 40, 41, 42, 43, -1, 3 * bs - 1, -1, 50, 51, 52, 53, 54, 55], device=DEV)
    _append_both(cache, qkv[:, 4:6], qkv[:, 6:8], slots, bs)
    assert _native.read_status(DEV) == _native.STATUS_BAD_SLOT
    odd = torch.randn(20 * H * D + 1, generator=g, device=DEV).half()[1:].view(20, H, D)          # 2 bytes off: copied by the call
    _append_both(cache, odd, odd.flip(0), torch.arange(20, device=DEV) + 17, bs)
    _append_both(cache, odd[:0], odd[:0], slots[:0], bs)
    before = cache.clone()
    quantize_and_scatter(odd, odd, cache, torch.full((20,), -1, device=DEV), bs)
    assert torch.equal(cache, before)


def test_append_refusals():
    x, slots, cache = torch.zeros(2, 4, 128, device=DEV, dtype=torch.float16), torch.arange(2, device=DEV), allocate_cache_8bit(2, 16, 4, DEV)
    bad = [dict(key=x[..., :96]), dict(value=x[:, :3]), dict(value=x.bfloat16()), dict(slot_mapping=slots[:1]), dict(block_size=32), dict(block_size=8),
           dict(cache=cache[:, :3].contiguous()), dict(cache=cache.view(torch.int8)), dict(key=x.transpose(0, 1)), dict(key=x.double(), value=x.double())]
    for change in bad:
        with pytest.raises(ValueError):
            quantize_and_scatter(**{**dict(key=x, value=x, cache=cache, slot_mapping=slots, block_size=16), **change})


# ---- attention over it ---------------------------------------------------------------------------------------
def _filled(g, lens, H, D, bs, spread=3):
    """A cache of random codes and scales (as the append kernel would leave them), tables whose unused entries are wild."""
    lens = torch.as_tensor(lens)
    blocks = (lens.clamp(min=0) + bs - 1) // bs
    n = max(1, int(blocks.sum()))
    cache = allocate_cache_8bit(n + 1, bs, H, DEV, D)
    codes, scales = codes_and_scales(cache, bs, D)
    x = torch.randn(codes.shape, generator=g, device=DEV) * 100
    codes.copy_(x.clamp(-448, 448).to(torch.float8_e4m3fn))
    scales.copy_(torch.exp2(torch.randint(-8 - spread, -8 + spread + 1, scales.shape, generator=g, device=DEV).float()))
    perm = torch.randperm(n + 1, generator=g, device=DEV).tolist()
    width = max(1, int(blocks.max()))
    tables = torch.full((len(lens), width), -(1 << 31) + 5, dtype=torch.int32)
    at = 0
    for i, b in enumerate(blocks.tolist()):
        tables[i, :b] = torch.tensor(perm[at:at + b], dtype=torch.int32)
        at += b
    # what lies behind the last token of a page is NaN in both, its scale is kept
    raw = codes.view(torch.uint8)
    for i, L in enumerate(lens.tolist()):
        if L > 0 and L % bs:
            b, off = int(tables[i, L // bs]), L % bs
            for p in range(bs // 16):
                raw[b, :, p, :, max(0, min(16, off - 16 * p)):] = 0x7f
    return cache, tables.to(DEV)


def _check_attention(g, lens, queries, Hq, H, D, bs, dtype, sm_scale=None, q_size=1.0, spread=3, width=0, **call):
    cache, tables = _filled(g, lens, H, D, bs, spread)
    if width > tables.shape[1]:                                             # launches are sized for the table where nothing else is said
        tables = torch.nn.functional.pad(tables, (0, width - tables.shape[1]), value=-9)
    T = sum(queries)
    q = (torch.randn(T, Hq, D, generator=g, device=DEV) * q_size).to(dtype)
    starts = np.concatenate([[0], np.cumsum(queries)])
    lens_t = torch.tensor(lens, **i32)
    if max(queries, default=1) > 1 or min(queries, default=1) < 1:
        call = dict(query_start_loc=torch.tensor(starts, **i32), max_query_len=max(max(queries), 1)) | call
    got = paged_attention_8bit(q, cache, tables, lens_t, bs, sm_scale=sm_scale, **call)
    codes, scales = _state(cache, bs, D)
    want, tol = S.attention(q.double().cpu().numpy(), codes, scales, tables.cpu().numpy(), lens, starts, bs,
                            1 / math.sqrt(D) if sm_scale is None else sm_scale, EPS[dtype])
    g64 = got.double().cpu().numpy()
    assert np.isfinite(g64).all()
    worst = (np.abs(g64 - want) / tol).max() if want.size else 0.0
    assert worst <= 1, worst
    return q, cache, tables, lens_t, got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,H,bs", [(1, 1, 16), (8, 1, 32), (10, 2, 16), (16, 1, 16), (6, 6, 32), (34, 2, 16)])
def test_single_queries(Hq, H, bs, D, dtype):
    """One query per sequence; lengths of nothing, one token, around pages, over the split of the work."""
    _check_attention(gen(Hq), [0, 1, 15, 16, 17, 31, 33, 64, 100, 257, 1000, -3, 2], [1] * 13, Hq, H, D, bs, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Hq,H", [(128, 8, 1), (64, 4, 4), (128, 28, 4)])
def test_one_long_sequence(D, Hq, H, dtype):
    _check_attention(gen(7), [5003], [1], Hq, H, D, 16, dtype, max_seq_len=5003)


@pytest.mark.parametrize("n,H,L", [(1, 1, 17), (1, 1, 300), (2, 4, 130), (5, 4, 600), (14, 5, 40), (19, 8, 33), (150, 1, 70)])
@pytest.mark.parametrize("G", [1, 8, 11])
def test_clusters_of_every_size(n, H, L, G):
    """Few items with clusters of 8, 4 and 2 CTAs, and of one, some of whose warps and CTAs have no page."""
    lens = [max(0, L - 13 * i) for i in range(n)]
    _check_attention(gen(n), lens, [1] * n, G * H, H, 128 if G > 1 else 64, 16, torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Hq,H,bs", [(128, 8, 2, 16), (64, 5, 1, 32), (128, 16, 1, 16), (128, 3, 3, 32)])
def test_several_queries_per_sequence(D, Hq, H, bs, dtype):
    """Speculated tokens and prompt chunks, causal among themselves; sequences without queries, and shorter than their queries."""
    _check_attention(gen(Hq), [40, 1, 300, 17, 0, 2, 64, 33], [4, 1, 7, 0, 3, 5, 64, 2], Hq, H, D, bs, dtype)


@pytest.mark.parametrize("queries,lens", [([130], [130]), ([200, 1, 77], [1000, 64, 77]), ([16, 129], [16, 400]), ([257, 64], [300, 64])])
@pytest.mark.parametrize("D,Hq,H", [(128, 8, 2), (64, 6, 1), (128, 1, 1)])
def test_prompt_chunks(queries, lens, D, Hq, H):
    _check_attention(gen(sum(queries)), lens, queries, Hq, H, D, 16, torch.bfloat16 if D == 128 else torch.float16)


# With wide tables the same calls take the persistent kernel: its shares then hold less than a page, parts of items, several items.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Hq,H,bs", [(128, 8, 1, 16), (64, 10, 2, 32), (128, 16, 1, 48), (64, 16, 1, 16), (128, 12, 6, 16)])
def test_wide_tables_single_queries(D, Hq, H, bs, dtype):
    _check_attention(gen(Hq), [0, 1, 15, 16, 17, 31, 33, 64, 100, 257, 1000, -3, 2], [1] * 13, Hq, H, D, bs, dtype, width=3000)


@pytest.mark.parametrize("lens", [[1], [0, 0, 0], [5003, 0, 0, 7], [16 * 2368 // 4], [16 * 2368 // 4 + 1, 1], [40] * 700, list(range(0, 1400, 3))])
@pytest.mark.parametrize("D,Hq,H", [(128, 8, 1), (64, 12, 4)])
def test_wide_tables_shares(lens, D, Hq, H):
    """Fewer pages than warps, one more than evenly shared, more sequences than entries of the prefix, shares of many items."""
    _check_attention(gen(len(lens)), lens, [1] * len(lens), Hq, H, D, 16, torch.float16, width=40000 // len(lens) + 1200)


@pytest.mark.parametrize("D,Hq,H,bs", [(128, 8, 2, 16), (64, 5, 1, 32), (128, 16, 1, 16), (128, 3, 3, 32)])
def test_wide_tables_several_queries(D, Hq, H, bs):
    lens, queries = [40, 1, 300, 17, 0, 2, 64, 33, 700], [4, 1, 7, 0, 3, 5, 6, 2, 8]
    _check_attention(gen(Hq), lens, queries, Hq, H, D, bs, torch.bfloat16, width=4000)


# Decodes, verified tokens and chunks in one call over many pages: two kernels share the sequences, by their number of query rows.
_MIXED = [1, 1, 0, 4, 130, 1, 2, 16, 17, 1, 5, 64, 1, 3, 1, 8, 1, 0, 33, 1]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Hq,H,bs", [(128, 8, 2, 16), (64, 16, 1, 32), (128, 3, 3, 48), (128, 12, 1, 16), (64, 34, 2, 16), (64, 8, 8, 16)])
def test_mixed_steps(D, Hq, H, bs, dtype):
    g = gen(Hq + H)
    lens = [n + int(x) for n, x in zip(_MIXED, torch.randint(0, 400, (len(_MIXED),), generator=torch.Generator().manual_seed(Hq)))]
    lens[0], lens[5], lens[8], lens[13] = 0, 1, 17, 2                       # no context, nothing at all, fewer tokens than queries
    _check_attention(g, lens, _MIXED, Hq, H, D, bs, dtype, width=40000 // (len(lens) * H * (bs // 16)) + 60)


@pytest.mark.parametrize("n", [2, 128, 129, 705, 1500])
def test_mixed_steps_of_many_sequences(n):
    """One chunk among decodes, at either end or inside; more sequences than are ranked, and than a CTA has threads."""
    for at in (0, n // 2, n - 1):
        queries, lens = [1] * n, [1 + (37 * i + at) % 70 for i in range(n)]
        queries[at], lens[at] = 150, 333
        _check_attention(gen(n), lens, queries, 8, 2, 64, 16, torch.bfloat16, width=40000 // (2 * n) + 60)


def test_mixed_steps_with_chunks_that_fill_the_gpu():
    _check_attention(gen(3), [40, 900, 33, 1000, 2, 0, 650], [1, 610, 2, 1, 2, 1, 40], 32, 8, 128, 16, torch.float16, width=700)


@pytest.mark.parametrize("width", [4, 2000])
def test_rows_behind_a_mixed_step(width):
    g = gen(21)
    queries, lens = [1, 70, 0, 1, 3], [50, 100, 20, 1, 33]
    q, cache, tables, lens_t, got = _check_attention(g, lens, queries, 8, 4, 128, 16, torch.float16, width=width)
    padded = torch.cat([q, torch.randn(9, 8, 128, generator=g, device=DEV).half()])
    starts = torch.tensor(np.concatenate([[0], np.cumsum(queries)]), **i32)
    new = paged_attention_8bit(padded, cache, tables, lens_t, 16, query_start_loc=starts, max_query_len=70)
    out = torch.full_like(padded, 7.0)
    paged_attention_8bit(padded, cache, tables, lens_t, 16, query_start_loc=starts, max_query_len=70, out=out)
    assert torch.equal(new[:75], out[:75]) and not new[75:].any() and (out[75:] == 7).all()
    assert torch.equal(new[:75], got)                                       # rows behind change nothing
    paged_attention_8bit(padded, cache, tables, lens_t, 16, query_start_loc=starts, max_query_len=65)
    assert _native.read_status(DEV) == _native.STATUS_TOO_LONG
    paged_attention_8bit(padded, cache, tables, lens_t + 16 * 3 * 2000, 16, query_start_loc=starts, max_query_len=70)
    assert _native.read_status(DEV) & _native.STATUS_BAD_BLOCK


def test_a_captured_mixed_step_follows_its_lengths():
    """Which kernel has which sequence is decided on the device: a replay with other lengths is that step's result.  Two graphs in turn, and a call
    on another stream between them."""
    g = gen(31)
    lens = [300, 90, 200, 64, 150, 500]
    cache, tables = _filled(g, lens, 2, 128, 16)
    tables = torch.nn.functional.pad(tables, (0, 3000), value=-9)
    q = torch.randn(120, 8, 128, generator=g, device=DEV).half()
    lens_t, starts = torch.tensor(lens, **i32), torch.zeros(7, **i32)
    call = dict(query_start_loc=starts, max_query_len=100)
    steps = [[1, 1, 100, 1, 1, 16], [64, 1, 0, 17, 1, 1], [1, 1, 1, 1, 1, 1], [0, 100, 2, 0, 18, 0]]
    cum = [torch.tensor(np.concatenate([[0], np.cumsum(s)]), **i32) for s in steps]
    starts.copy_(cum[0])
    paged_attention_8bit(q, cache, tables, lens_t, 16, **call)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(paged_attention_8bit(q, cache, tables, lens_t, 16, **call))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for c in cum:
        starts.copy_(c)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            want = paged_attention_8bit(q, cache, tables, lens_t, 16, query_start_loc=c, max_query_len=100)
        for graph, out in zip(graphs, outs):
            out.fill_(3)
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        torch.cuda.synchronize()


def test_negative_and_zero_scales():
    for width in (0, 9000):
        _check_attention(gen(5), [300, 40], [1, 1], 8, 2, 128, 16, torch.float16, sm_scale=-0.05, width=width)
        _check_attention(gen(6), [300, 40], [1, 1], 8, 2, 128, 16, torch.bfloat16, sm_scale=0.0, width=width)


def test_scores_of_any_size():
    """Scores of thousands (one key takes all), scales of the pages far apart, queries near the ends of their types."""
    _check_attention(gen(1), [300, 40], [1, 1], 8, 2, 128, 16, torch.float16, q_size=30.0, spread=0, sm_scale=0.02)
    _check_attention(gen(2), [300, 40], [1, 1], 8, 2, 128, 16, torch.bfloat16, spread=40, sm_scale=2.0 ** -45)
    _check_attention(gen(3), [300, 40], [1, 1], 8, 2, 128, 16, torch.bfloat16, q_size=1e30, sm_scale=1e-32)
    _check_attention(gen(4), [300, 40], [1, 1], 8, 2, 128, 16, torch.bfloat16, q_size=1e-30, sm_scale=1e28)


@pytest.mark.parametrize("width,n", [(0, 1), (9000, 1), (0, 40)])
def test_values_of_very_different_sizes(width, n):
    """Pages whose values are 2^24 apart: the small ones count for the denominator, whatever fp16 holds of their weights."""
    for dtype, spread, scale in ((torch.float16, 9, 3e-5), (torch.bfloat16, 30, 2.0 ** -42)):
        _check_attention(gen(n), [300, 140], [n, n], 8, 2, 128, 16, dtype, spread=spread, sm_scale=scale, width=width)


@pytest.mark.parametrize("width,n", [(0, 1), (9000, 1), (0, 40)])
def test_a_token_that_takes_all_is_exact(width, n):
    """One key is the query's, the others are far: the output is that token's value, rounded once."""
    g = gen(31)
    H, D, bs, L = 2, 128, 16, 200
    cache, tables = _filled(g, [L], H, D, bs)
    codes, scales = codes_and_scales(cache, bs)
    scales[..., 0] = 1.0
    q = torch.zeros(n, 4 * H, D, device=DEV, dtype=torch.float16)
    raw = codes.view(torch.uint8)
    raw[:, :, :, 0] = 0                                                     # all keys zero but that of token 100, dim 7
    b, at = int(tables[0, 100 // bs]), 100 % bs
    raw[b, :, 0, 0, at, 7] = 0x7e
    q[..., 7] = 30.0
    if width:
        tables = torch.nn.functional.pad(tables, (0, width - tables.shape[1]))
    more = {} if n == 1 else dict(query_start_loc=torch.tensor([0, n], **i32), max_query_len=n)
    got = paged_attention_8bit(q, cache, tables, torch.tensor([L], **i32), bs, sm_scale=1.0, **more)
    want = (codes[b, :, 0, 1, at].float() * scales[b, :, 0, 1][:, None]).half()
    assert torch.equal(got, want.repeat_interleave(4, 0).expand(n, -1, -1))


def test_nan_reaches_what_sees_it_and_nothing_else():
    """A NaN value in a token that some queries of a chunk see and earlier ones do not; a NaN key."""
    g = gen(11)
    cache, tables = _filled(g, [60, 60], 1, 128, 16)
    codes, _ = codes_and_scales(cache, 16)
    raw = codes.view(torch.uint8)
    raw[int(tables[0, 3]), 0, 0, 1, 5, 77] = 0xff                          # value of token 53, dim 77
    raw[int(tables[1, 3]), 0, 0, 0, 9, 3] = 0x7f                           # key of token 57
    q = torch.randn(40, 4, 128, generator=g, device=DEV).half()
    starts, lens = torch.tensor([0, 20, 40], **i32), torch.tensor([60, 60], **i32)
    got = paged_attention_8bit(q, cache, tables, lens, 16, query_start_loc=starts, max_query_len=20)
    c, s = _state(cache, 16, 128)
    want, tol = S.attention(q.double().cpu().numpy(), c, s, tables.cpu().numpy(), [60, 60], [0, 20, 40], 16, 128 ** -0.5, EPS[torch.float16])
    g64 = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(g64), np.isnan(want))
    assert np.isnan(g64[13:20, :, 77]).all() and not np.isnan(g64[:13]).any() and np.isnan(g64[37:]).all()
    fine = ~np.isnan(want)
    assert (np.abs(g64 - want)[fine] <= tol[fine]).all()


def test_rows_behind_the_last_sequence():
    g = gen(12)
    cache, tables = _filled(g, [20, 30], 1, 64, 16)
    q = torch.randn(9, 2, 64, generator=g, device=DEV).half()
    starts, lens = torch.tensor([0, 2, 5], **i32), torch.tensor([20, 30], **i32)
    out = torch.full_like(q, 7.0)
    res = paged_attention_8bit(q, cache, tables, lens, 16, query_start_loc=starts, max_query_len=3, out=out)
    assert res is out and (out[5:] == 7).all()
    new = paged_attention_8bit(q, cache, tables, lens, 16, query_start_loc=starts, max_query_len=3)
    assert torch.equal(new[:5], out[:5]) and not new[5:].any()
    none = paged_attention_8bit(q, cache, tables, lens, 16, query_start_loc=starts[:1], max_query_len=3)
    assert not none.any()
    few = paged_attention_8bit(q, cache, tables, lens, 16, query_start_loc=starts, max_query_len=2)
    assert _native.read_status(DEV) == _native.STATUS_TOO_LONG and torch.isfinite(new).all() and few.shape == q.shape


def test_bad_tables_and_lengths_are_cut_and_flagged():
    g = gen(13)
    cache, tables = _filled(g, [64, 64, 64], 2, 128, 16)
    cache.bitwise_and_(0x77)                                                # no NaN wherever it reads
    q = torch.randn(3, 4, 128, generator=g, device=DEV).bfloat16()
    bad = tables.clone()
    bad[0, 2], bad[1, 1] = -1, 1 << 30
    clamped = bad.clamp(0, cache.shape[0] - 1)
    lens = torch.tensor([64, 64, 64], **i32)
    got = paged_attention_8bit(q, cache, bad, lens, 16)
    assert _native.read_status(DEV) == _native.STATUS_BAD_BLOCK
    assert torch.equal(got, paged_attention_8bit(q, cache, clamped, lens, 16))
    got = paged_attention_8bit(q, cache, tables, torch.tensor([(1 << 31) - 1, 64, 1 << 30], **i32), 16)
    assert _native.read_status(DEV) == _native.STATUS_BAD_BLOCK
    assert torch.equal(got, paged_attention_8bit(q, cache, tables, lens, 16))
    wild = torch.tensor([2, -7, 1 << 30, 3], **i32)                         # offsets that are none: nothing outside q is touched
    paged_attention_8bit(q, cache, tables, lens, 16, query_start_loc=wild, max_query_len=2)
    _native.read_status(DEV)


def test_a_cache_beyond_32_bits():
    """Pages further than 2^32 bytes into the cache."""
    D, H, bs = 128, 8, 32
    blocks = (1 << 32) // (H * 2 * 4128) + 3000
    cache = torch.empty(blocks, H, 2 * 4128, dtype=torch.uint8, device=DEV)
    g = gen(14)
    table = torch.tensor([[blocks - 1, 0, blocks - 2, 66000]], **i32)
    slots = (table[0].long()[:, None] * bs + torch.arange(bs, device=DEV)).view(-1)[:100]
    kv = torch.randn(2, 100, H, D, generator=g, device=DEV).half()
    quantize_and_scatter(*kv, cache, slots, bs)
    q = torch.randn(1, 16, D, generator=g, device=DEV).half()
    got = paged_attention_8bit(q, cache, table, torch.tensor([100], **i32), bs)
    small = allocate_cache_8bit(4, bs, H, DEV)
    quantize_and_scatter(*kv, small, torch.arange(100, device=DEV), bs)
    want = paged_attention_8bit(q, small, torch.arange(4, **i32)[None], torch.tensor([100], **i32), bs)
    assert torch.equal(got, want)


def test_attention_refusals():
    q, cache = torch.zeros(2, 8, 128, device=DEV, dtype=torch.float16), allocate_cache_8bit(4, 16, 2, DEV)
    tables, lens = torch.zeros(2, 2, **i32), torch.ones(2, **i32)
    starts = torch.tensor([0, 1, 2], **i32)
    bad = [dict(q=q.float()), dict(q=q[..., :96].contiguous()), dict(q=q[:, :7].contiguous()), dict(block_size=32), dict(block_size=0), dict(seq_lens=lens[:1]),
           dict(block_tables=tables[:1]), dict(max_query_len=2), dict(query_start_loc=starts, max_query_len=0), dict(cache=cache[:0]),
           dict(block_tables=tables[0]), dict(out=q[:1]), dict(out=q.bfloat16()), dict(cache=cache.view(torch.int8))]
    for change in bad:
        with pytest.raises(ValueError):
            paged_attention_8bit(**{**dict(q=q, cache=cache, block_tables=tables, seq_lens=lens, block_size=16), **change})
    with pytest.raises(RuntimeError, match="no autograd"):
        paged_attention_8bit(q.requires_grad_(), cache, tables, lens, 16, out=torch.zeros_like(q))


# ---- step tables -----------------------------------------------------------------------------------------------
def _check_plan(query, context, width, free, count, bs, rows):
    g = torch.Generator().manual_seed(len(query))
    tables = torch.randint(0, 1000, (len(query), width), generator=g, dtype=torch.int32)
    want = S.plan(query, context, tables.numpy(), free, count, bs, rows)
    t = tables.to(DEV)
    args = (torch.tensor(query, **i32), torch.tensor(context, **i32), t, torch.tensor(free, **i32), torch.tensor([count], **i32), bs, rows)
    for _ in range(2):                                                      # a repeated call gives the same tables
        plan = plan_step(*args)
        assert _native.read_status(DEV) == want[6]
        for name, got, w in zip(("slots", "positions", "lens", "starts", "count", "tables"),
                                (plan.slot_mapping, plan.positions, plan.seq_lens, plan.query_start_loc, plan.free_count[0], t), want):
            assert np.array_equal(got.cpu().numpy(), w), name
    return plan, t


@pytest.mark.parametrize("n,bs", [(1, 16), (5, 16), (64, 32), (700, 16), (2049, 16), (5000, 32)])
def test_plan_of_mixed_steps(n, bs):
    r = np.random.default_rng(n)
    query, context = r.integers(0, 5, n), r.integers(0, 200, n)
    query[r.random(n) < 0.02] = 150
    context[r.random(n) < 0.1] = 0
    total = int(query.sum())
    free = r.permutation(total // bs + 2 * n)
    _check_plan(query, context, 350 // bs + 1, free, len(free), bs, total)
    _check_plan(query, context, 350 // bs + 1, free, len(free), bs, total + 37)              # rows behind the last request
    _check_plan(query, context, 350 // bs + 1, free, n // 3, bs, total + 1)                  # not enough blocks
    _check_plan(query, context, 200 // bs, free, len(free), bs, total)                       # tables too narrow for some
    _check_plan(query, context, 350 // bs + 1, free, len(free), bs, total // 2)              # rows do not suffice


def test_plan_at_its_edges():
    _check_plan([1], [0], 1, [5], 1, 16, 1)
    _check_plan([0, 0], [16, 17], 2, [5], 1, 16, 0)
    _check_plan([-4, 3, -1], [5, -2, 16], 2, [5, 6], 2, 16, 5)
    _check_plan([1, 1], [16, 15], 2, [], 0, 16, 2)
    _check_plan([1, 1], [16, 15], 2, [7], 9, 16, 2)                                          # a count beyond the stack
    _check_plan([100000], [3], 100003 // 16 + 1, list(range(6300)), 6300, 16, 100000)
    _check_plan([2 ** 30, 5], [2 ** 30 + 2 ** 29, 3], 3, [1, 2, 3], 3, 16, 8)
    _check_plan([], [], 3, [1, 2, 3], 3, 16, 4)


@pytest.mark.parametrize("n,bs", [(1, 16), (40, 32), (3000, 16)])
def test_release(n, bs):
    r = np.random.default_rng(n)
    ended, context = r.random(n) < 0.5, r.integers(0, 300, n)
    ended[0] = True
    tables = r.integers(0, 100000, (n, 300 // bs + 1)).astype(np.int32)
    need = int((-(-context // bs))[ended].sum())
    for size, count in ((need + 10, 10), (need + 3, 0), (max(need // 2, 1), 1)):
        free = r.integers(0, 9, size)
        want = S.release(ended, context, tables, free, count, bs)
        stack = torch.tensor(free, **i32)
        lens, new = release_blocks(torch.tensor(ended, device=DEV), torch.tensor(context, **i32), torch.tensor(tables, **i32), stack,
                                   torch.tensor([count], **i32), bs)
        assert _native.read_status(DEV) == (0 if need + count <= size else _native.STATUS_TOO_LONG)
        assert np.array_equal(lens.cpu().numpy(), want[0]) and int(new) == want[1] and np.array_equal(stack.cpu().numpy(), want[2])


def test_plan_refusals():
    v, t, c = torch.ones(2, **i32), torch.zeros(2, 4, **i32), torch.ones(1, **i32)
    bad = [dict(query_lens=v.long()), dict(context_lens=v[:1]), dict(block_tables=t[:1]), dict(block_tables=t.long()), dict(free_count=v), dict(block_size=0),
           dict(num_rows=-1), dict(block_tables=t.t()), dict(free_blocks=t)]
    for change in bad:
        with pytest.raises(ValueError):
            plan_step(**{**dict(query_lens=v, context_lens=v, block_tables=t, free_blocks=v, free_count=c, block_size=16, num_rows=2), **change})
    ok = dict(ended=v.bool(), context_lens=v, block_tables=t, free_blocks=v, free_count=c, block_size=16)
    for change in [dict(ended=v), dict(ended=v.bool()[:1]), dict(free_blocks=v.long()), dict(block_size=-1)]:
        with pytest.raises(ValueError):
            release_blocks(**{**ok, **change})


# ---- together ------------------------------------------------------------------------------------------------------
def test_a_serving_loop():
    """Requests come, run and end over several steps: tables, rotary positions, cache and attention, against attention over the
    rotated keys and values as they were given (the cache's e4m3 values are within 2^-4 of them)."""
    D, Hq, H, bs, n, blocks = 128, 8, 2, 16, 6, 40
    g = gen(21)
    table = make_rotary_table(D, 1024, device=DEV)
    cache = allocate_cache_8bit(blocks, bs, H, DEV)
    tables, free, count = torch.zeros(n, 16, **i32), torch.randperm(blocks, generator=g, device=DEV).to(torch.int32), torch.tensor([blocks], **i32)
    context = torch.zeros(n, **i32)
    history = [[] for _ in range(n)]
    for step in range(8):
        new = [(37, 5, 16, 1, 0, 90), (1,) * 6, (1, 1, 1, 1, 20, 1), (4, 1, 2, 1, 1, 3)][min(step, 3)]
        T = sum(new) + 2                                                     # two rows of padding
        plan = plan_step(torch.tensor(new, **i32), context, tables, free, count, bs, T)
        qkv = torch.randn(T, Hq + 2 * H, D, generator=g, device=DEV).half()
        q, k = rotary_embedding(qkv[:, :Hq], qkv[:, Hq:Hq + H], plan.positions, table)
        v = qkv[:, Hq + H:]
        quantize_and_scatter(k, v, cache, plan.slot_mapping, bs)
        out = paged_attention_8bit(q, cache, tables, plan.seq_lens, bs, query_start_loc=plan.query_start_loc, max_query_len=max(new))
        assert not out[T - 2:].any()
        starts = plan.query_start_loc.tolist()
        for i in range(n):
            a, b = starts[i], starts[i + 1]
            history[i] += [(k[r], v[r]) for r in range(a, b)]
            if a == b:
                continue
            assert int(plan.seq_lens[i]) == len(history[i])
            K, V = (torch.stack(x).float().repeat_interleave(Hq // H, 1) for x in zip(*history[i]))
            s = torch.einsum("jhd,khd->hjk", q[a:b].float(), K) * D ** -0.5
            hidden = torch.arange(len(K), device=DEV) > torch.arange(len(K) - (b - a), len(K), device=DEV)[:, None]
            want = torch.einsum("hjk,khd->jhd", s.masked_fill(hidden, -math.inf).softmax(-1), V)
            # values off by at most 2^-4, weights by what scores are off: |q| |k| 2^-4 sm_scale at random signs
            assert (out[a:b].float() - want).norm() <= 0.08 * want.norm()
        context, count = plan.seq_lens, plan.free_count
        if step in (3, 5):
            ended = torch.tensor([True, False, False, step == 5, False, True], device=DEV)
            context, count = release_blocks(ended, context, tables, free, count, bs)
            history = [[] if e else h for e, h in zip(ended.tolist(), history)]
            held = int(((context + bs - 1) // bs).sum())
            assert int(count) == blocks - held
            alive = torch.cat([free[:int(count)]] + [tables[i, :(int(context[i]) + bs - 1) // bs] for i in range(n)])
            assert alive.sort().values.tolist() == list(range(blocks))


def test_captured_and_replayed():
    """A whole step in a CUDA graph, replayed with other lengths and inputs; a second graph beside it; another stream."""
    D, Hq, H, bs, n = 128, 16, 2, 16, 5
    g = gen(22)
    table = make_rotary_table(D, 4096, device=DEV)
    free, count = torch.arange(200, **i32), torch.tensor([200], **i32)
    # every request has blocks of its own for whatever context it is given below; new ones come from the stack
    query, context = torch.ones(n, **i32), torch.tensor([0, 15, 16, 300, 1000], **i32)
    tables = torch.arange(200, 200 + 80 * n, **i32).view(n, 80)
    held = tables.clone()
    cache = allocate_cache_8bit(200 + 80 * n, bs, H, DEV)
    total = cache.shape[0] * bs
    quantize_and_scatter(*torch.randn(2, total, H, D, generator=g, device=DEV).half(), cache, torch.arange(total, device=DEV), bs)
    qkv = torch.randn(n, Hq + 2 * H, D, generator=g, device=DEV).half()

    def step():
        plan = plan_step(query, context, tables, free, count, bs, n)
        q, k = rotary_embedding(qkv[:, :Hq], qkv[:, Hq:Hq + H], plan.positions, table)
        quantize_and_scatter(k, qkv[:, Hq + H:], cache, plan.slot_mapping, bs)
        return paged_attention_8bit(q, cache, tables, plan.seq_lens, bs, max_seq_len=1280)

    start = cache.clone()

    def reset():
        cache.copy_(start)
        tables.copy_(held)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for k in range(3):
        qkv.normal_(generator=g)
        context.copy_(torch.tensor([k, 15 + k, 16, 300 - k, 1000 + 8 * k], **i32))
        reset()
        want, state = step().clone(), cache.clone()
        reset()
        graphs[k % 2].replay()
        assert torch.equal(outs[k % 2], want) and torch.equal(cache, state)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        reset()
        other = step()
    side.synchronize()
    assert torch.equal(other, want)


def test_compiled_and_traced_operators():
    """The registered operators agree with the direct calls, and their shapes are known without running them."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    g = gen(23)
    cache, tables = _filled(g, [20, 30], 1, 64, 16)
    q = torch.randn(2, 4, 64, generator=g, device=DEV).half()
    lens, table = torch.tensor([20, 30], **i32), make_rotary_table(64, 64, device=DEV)
    direct = paged_attention_8bit(q, cache, tables, lens, 16)
    assert torch.equal(torch.ops.tq_b200.attend8_paged(q, cache, tables, lens, None, 0.125, 16, 1, 0), direct)
    a, b = torch.ops.tq_b200.rotary(q, None, lens, table, False, False)
    assert torch.equal(a, rotary_embedding(q, None, lens, table)[0]) and b.numel() == 0
    one, other = cache.clone(), cache.clone()
    slots = torch.tensor([3, 20], device=DEV)
    torch.ops.tq_b200.quantize8_paged(q[:, :1], q[:, 1:2], one, slots, 16)
    version = other._version
    quantize_and_scatter(q[:, :1], q[:, 1:2], other, slots, 16)
    assert torch.equal(one, other) and other._version > version
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        f = mode.from_tensor
        assert torch.ops.tq_b200.attend8_paged(f(q), f(cache), f(tables), f(lens), None, 0.125, 16, 1, 0).shape == q.shape
        assert [t.shape for t in torch.ops.tq_b200.plan_step(f(lens), f(lens), f(tables), f(lens), f(lens[:1]), 16, 9)] == [(9,), (9,), (2,), (3,), (1,)]
    with pytest.raises(RuntimeError):
        rotary_embedding(q.float().requires_grad_(), None, lens, table)[0].sum().backward()
