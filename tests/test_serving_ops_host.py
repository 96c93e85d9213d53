"""Host side of the operators around attention: rotary tables, views of the 8-bit cache, what the launchers refuse.  No GPU."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import serving_oracle as S
from turboquant.kernels import _native
from turboquant.kernels.block_plan import plan_step, release_blocks
from turboquant.kernels.paged_8bit import (allocate_cache_8bit, cache_shape_8bit, codes_and_scales, page_bytes_8bit,
                                           paged_attention_8bit, quantize_and_scatter)
from turboquant.kernels.rotary import make_rotary_table, rotary_embedding

NULL = ctypes.c_void_p(0)


def at(a):
    return ctypes.c_void_p(0x10000 + a)


# ---- the oracle's number format agrees with torch's ----------------------------------------------
def test_e4m3_of_the_oracle_is_torchs():
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes.copy()).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(S.e4m3_decode(codes), want)
    x = np.concatenate([np.random.default_rng(0).normal(size=4000) * 10.0 ** np.linspace(-4, 2.6, 4000), want[np.isfinite(want)],
                        (want[1:127] + want[:126]) / 2]).astype(np.float32)
    got = torch.from_numpy(x).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    np.testing.assert_array_equal(S.e4m3_encode(x.astype(np.float64)), got)


# ---- rotary tables -------------------------------------------------------------------------------
def _table_angles(table):
    half = table.shape[1] // 2
    return table[:, :half].double(), table[:, half:].double()


@pytest.mark.parametrize("dim,base", [(2, 10000.0), (20, 10000.0), (128, 500000.0)])
def test_plain_table(dim, base):
    table = make_rotary_table(dim, 200000, base)
    pos = np.array([0, 1, 77, 65535, 65536, 199999])
    angle = pos[:, None] * base ** (-np.arange(0, dim, 2) / dim)
    cos, sin = _table_angles(table[pos])
    # one rounding to fp32; the angles themselves, up to 2e5, are good to 2e5 * 2^-53 and the power's last bits
    np.testing.assert_allclose(cos.numpy(), np.cos(angle), atol=2.0 ** -24, rtol=0)
    np.testing.assert_allclose(sin.numpy(), np.sin(angle), atol=2.0 ** -24, rtol=0)


def _angles_at_1(table):
    cos, sin = _table_angles(table[1:2])
    return torch.atan2(sin, cos)[0], torch.hypot(cos, sin)[0]


def test_scaled_tables():
    dim, base, P = 64, 10000.0, 256
    f = base ** (-np.arange(0, dim, 2) / dim)
    linear, size = _angles_at_1(make_rotary_table(dim, P, base, {"rope_type": "linear", "factor": 4.0}))
    np.testing.assert_allclose(linear.numpy(), f / 4, rtol=1e-6)
    np.testing.assert_allclose(size.numpy(), 1, rtol=1e-6)

    llama, _ = _angles_at_1(make_rotary_table(dim, P, base, {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                                                             "original_max_position_embeddings": 8192}))
    for got, x in zip(llama.tolist(), f):
        wavelength = 2 * math.pi / x
        if wavelength < 8192 / 4:
            want = x
        elif wavelength > 8192:
            want = x / 8
        else:
            smooth = (8192 / wavelength - 1) / 3
            want = (1 - smooth) * x / 8 + smooth * x
        assert abs(got - want) <= 1e-6 * want

    yarn, size = _angles_at_1(make_rotary_table(dim, P, base, {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}))
    low = math.floor(dim * math.log(4096 / (32 * 2 * math.pi)) / (2 * math.log(base)))
    high = math.ceil(dim * math.log(4096 / (2 * math.pi)) / (2 * math.log(base)))
    np.testing.assert_allclose(yarn[:low + 1].numpy(), f[:low + 1], rtol=1e-6)                # fast pairs stay
    np.testing.assert_allclose(yarn[high:].numpy(), f[high:] / 16, rtol=1e-6)                 # slow ones are stretched
    assert all(f[i] / 16 < yarn[i] < f[i] for i in range(low + 1, high))
    np.testing.assert_allclose(size.numpy(), 0.1 * math.log(16) + 1, rtol=1e-6)

    # beyond the trained length the slowest pair turns 1 / grown as fast, within it nothing changes
    spec = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 512}
    same, _ = _angles_at_1(make_rotary_table(dim, 512, base, spec))
    np.testing.assert_allclose(same.numpy(), f, rtol=1e-6)
    longer, _ = _angles_at_1(make_rotary_table(dim, 2048, base, spec))
    np.testing.assert_allclose(longer.numpy(), (base * (2 * 2048 / 512 - 1) ** (dim / (dim - 2))) ** (-np.arange(0, dim, 2) / dim), rtol=1e-6)


def test_tables_that_are_refused():
    for args in ((3, 16), (0, 16), (64, 0)):
        with pytest.raises(ValueError):
            make_rotary_table(*args)
    with pytest.raises(ValueError, match="not known"):
        make_rotary_table(64, 16, scaling={"rope_type": "spiral", "factor": 2.0, "original_max_position_embeddings": 8})
    with pytest.raises(ValueError, match="at least 1"):
        make_rotary_table(64, 16, scaling={"rope_type": "linear", "factor": 0.5})


# ---- the cache's layout ----------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
def test_cache_views(dim):
    assert page_bytes_8bit(dim) == 32 * dim + 32 and cache_shape_8bit(3, 32, 2, dim) == (3, 2, 2 * (32 * dim + 32))
    cache = allocate_cache_8bit(3, 32, 2, "cpu", dim)
    codes, scales = codes_and_scales(cache, 32, dim)
    assert codes.shape == (3, 2, 2, 2, 16, dim) and scales.shape == (3, 2, 2, 2)
    codes.view(torch.uint8)[1, 0, 1, 1, 5, 7] = 42
    scales[1, 0, 1, 1] = 0.5
    page = cache[1, 0].view(2, -1)[1]
    assert page[16 * dim + 5 * dim + 7] == 42 and page[32 * dim + 4:32 * dim + 8].view(torch.float32) == 0.5
    assert int((cache != 0).sum()) == 2                                  # 0.5 is 0x3f000000


def test_cache_shapes_that_are_refused():
    with pytest.raises(ValueError, match="multiple of 16"):
        cache_shape_8bit(1, 24, 1)
    with pytest.raises(ValueError, match="head_dim"):
        page_bytes_8bit(96)
    with pytest.raises(ValueError, match="does not match"):
        codes_and_scales(torch.zeros(1, 1, 100, dtype=torch.uint8), 16)


# ---- the C interface ---------------------------------------------------------------------------------
def _rotary(L, q=at(0), k=at(0), qo=at(0), ko=at(0), dtype=0, strides=(256, 64) * 4, pos=at(0), wide=1, table=at(0), P=8, T=4, hq=4, hk=2, D=64, R=64,
            inter=0):
    st = (ctypes.c_int64 * 8)(*strides)
    return L.tq_rotary(q, k, qo, ko, dtype, st, pos, wide, table, P, T, hq, hk, D, R, inter, 0, NULL, NULL)


def test_rotary_refuses_without_touching_a_gpu():
    L = _native.lib()
    assert _rotary(L, T=0) == 0 and _rotary(L, hq=0, hk=0) == 0
    assert _rotary(L, q=NULL) == _rotary(L, ko=NULL) == _rotary(L, pos=NULL) == _rotary(L, table=NULL) == -1
    assert _rotary(L, R=65) == _rotary(L, R=66) == _rotary(L, R=0) == _rotary(L, P=0) == _rotary(L, T=-1) == -1
    assert _rotary(L, q=at(1)) == _rotary(L, pos=at(4)) == _rotary(L, wide=0, pos=at(2)) == _rotary(L, table=at(2)) == -1
    assert _rotary(L, q=at(2), inter=1) == -1                             # pairs that do not start on their own size
    assert _rotary(L, dtype=3) == -2


def test_cache8_calls_refuse_without_touching_a_gpu():
    L = _native.lib()

    def quantize(key=at(0), value=at(0), dtype=0, st=(256, 128, 256, 128), cache=at(0), blocks=4, bs=16, slots=at(0), T=4, H=2, D=128):
        return L.tq_quantize8_paged(key, value, dtype, *st, cache, blocks, bs, slots, T, H, D, NULL, NULL)

    assert quantize(T=0) == quantize(blocks=0) == quantize(H=0) == 0
    assert quantize(key=NULL) == quantize(cache=NULL) == quantize(slots=NULL) == quantize(T=-1) == -1
    assert quantize(key=at(8)) == quantize(cache=at(8)) == quantize(slots=at(4)) == quantize(st=(256, 124, 256, 128)) == -1
    assert quantize(D=96) == quantize(bs=24) == quantize(bs=0) == quantize(dtype=3) == -2
    assert L.tq_cache8_page_bytes(256) == -2

    def attend(out=at(0), q=at(0), dtype=0, cache=at(0), blocks=4, bs=16, tables=at(0), lens=at(0), starts=NULL, ws=NULL, nb=0, T=2, ns=2, hq=8, hk=2, D=128,
               most=1, pages=4):
        return L.tq_attend8_paged(out, q, dtype, cache, blocks, bs, tables, 1, lens, starts, 1.0, ws, nb, NULL, T, ns, hq, hk, D, most, pages, 0, NULL)

    assert attend(T=0, ns=0) == attend(T=4, ns=0, starts=at(0)) == 0
    assert attend(q=NULL) == attend(tables=NULL) == attend(blocks=0) == attend(hq=7) == attend(most=0) == attend(T=1) == attend(most=2) == -1
    assert attend(q=at(8)) == attend(out=at(8)) == attend(cache=at(8)) == -1
    assert attend(dtype=2) == attend(D=96) == attend(bs=8) == attend(pages=(1 << 27)) == -2
    assert attend(T=1, ns=1, pages=20000) == -4                             # shared out over the GPU, and no workspace
    need = L.tq_attend8_workspace_bytes(1, 1, 8, 2, 128, 1, 20000)
    assert need > 0 and L.tq_attend8_workspace_bytes(0, 0, 8, 2, 128, 1, 256) == 0
    assert L.tq_attend8_workspace_bytes(1, 1, 8, 3, 128, 1, 256) == -1 and L.tq_attend8_workspace_bytes(1, 1, 8, 2, 96, 1, 256) == -2


def test_plan_calls_refuse_without_touching_a_gpu():
    L = _native.lib()
    plan = lambda q=at(0), tables=at(0), free=at(0), count=at(0), slots=at(0), n=2, width=4, F=8, bs=16, rows=4: L.tq_plan_step(
        q, at(0), tables, width, free, count, slots, at(0), at(0), at(0), at(0), NULL, n, width, F, bs, rows, NULL)
    assert plan(q=NULL) == plan(tables=NULL) == plan(free=NULL) == plan(count=NULL) == plan(slots=NULL) == plan(n=-1) == plan(rows=-1) == plan(bs=0) == -1
    assert plan(n=1 << 25) == -2
    free = lambda ended=at(0), count=at(0), n=2, bs=16: L.tq_release_blocks(ended, at(0), at(0), 4, at(0), count, at(0), at(0), NULL, n, 4, 8, bs, NULL)
    assert free(ended=NULL) == free(count=NULL) == free(n=-1) == free(bs=0) == -1


# ---- Python refuses CPU tensors and shapes that do not fit ----------------------------------------------
def test_no_cpu_path():
    x, i32 = torch.zeros(2, 4, 128, dtype=torch.float16), dict(dtype=torch.int32)
    cache = allocate_cache_8bit(2, 16, 4, "cpu")
    with pytest.raises(RuntimeError, match="no CPU path"):
        rotary_embedding(x, x, torch.arange(2), make_rotary_table(128, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        quantize_and_scatter(x, x, cache, torch.arange(2), 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        paged_attention_8bit(x, cache, torch.zeros(2, 1, **i32), torch.ones(2, **i32), 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        plan_step(torch.ones(2, **i32), torch.ones(2, **i32), torch.zeros(2, 4, **i32), torch.arange(4, **i32), torch.ones(1, **i32), 16, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        release_blocks(torch.ones(2, dtype=torch.bool), torch.ones(2, **i32), torch.zeros(2, 4, **i32), torch.arange(4, **i32), torch.ones(1, **i32), 16)
    with pytest.raises(ValueError, match="int32 or int64"):
        rotary_embedding(x, x, torch.zeros(2), make_rotary_table(128, 4))


# ---- the oracle's tables by hand ---------------------------------------------------------------------
def test_plan_of_the_oracle_by_hand():
    tables = np.full((3, 3), 9)
    slots, pos, lens, starts, count, tables, status = S.plan([2, 1, 3], [3, 4, 0], tables, [10, 11, 12, 13], 4, 4, 8)
    # request 0: position 3 in its block 9, 4 in a new one; 1: a new block; 2: a new block
    assert slots.tolist() == [9 * 4 + 3, 13 * 4, 12 * 4, 11 * 4, 11 * 4 + 1, 11 * 4 + 2, -1, -1]
    assert pos.tolist() == [3, 4, 4, 0, 1, 2, 0, 0] and lens.tolist() == [5, 5, 3] and starts.tolist() == [0, 2, 3, 6]
    assert count == 1 and status == 0 and tables.tolist() == [[9, 13, 9], [9, 12, 9], [11, 9, 9]]
    lens, count, free = S.release([True, False, True], [5, 5, 3], tables, [10, 0, 0, 0, 0], 1, 4)
    assert lens.tolist() == [0, 5, 0] and count == 4 and free.tolist() == [10, 9, 13, 11, 0]


# ---- the engine's hook ---------------------------------------------------------------------------------
def test_eight_bit_backend():
    pytest.importorskip("vllm")
    from turboquant.integration import tq_b200_backend as B
    backend = B.TurboQuantB200EightBitBackend
    assert backend.get_impl_cls() is B.TurboQuantB200EightBitImpl and backend.get_supported_head_sizes() == [64, 128]
    assert backend.get_kv_cache_shape(5, 32, 2, 128) == (5, 2, 2 * 4128) and backend.get_name() == "CUSTOM"
    assert B.TurboQuantB200Backend.get_impl_cls() is B.TurboQuantB200Impl
    with pytest.raises(NotImplementedError):
        B.TurboQuantB200EightBitImpl(8, 128, 1.0, 2, sliding_window=64)


# ---- rows that are not where the kernel can read them -----------------------------------------------------
def test_rows_are_copied_once_where_they_have_to_be():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Copies(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(func.__name__)
            return func(*args, **(kwargs or {}))

    flat = torch.arange(5 * 3 * 128 + 8, dtype=torch.float16)
    for t, copied in ((flat[:-8].view(5, 3, 128), 0), (flat[1:-7].view(5, 3, 128), 1), (flat[:5 * 387].as_strided((5, 3, 128), (385, 128, 1)), 1),
                      (flat[:-8].view(5, 3, 128)[:, :2, :64], 0)):
        with Copies() as seen:
            got = _native._with_aligned_rows(t)
        assert torch.equal(got, t) and len(seen.names) == copied and (copied or got is t)
        assert got.data_ptr() % 16 == 0 and all(s * 2 % 16 == 0 for s in got.stride()[:2]) and got.stride(2) == 1
