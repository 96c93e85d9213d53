"""The 8-bit attention implementation on a GPU, with hand-built layer and metadata objects: prompts, decodes, steps that mix them and
prompts that continue cached context, against attention over the keys and values as they were given."""
import math
from types import SimpleNamespace

import pytest
import torch

from turboquant.integration import tq_b200_backend as B
from turboquant.kernels import _native

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("D,Hq,H,bs,dtype", [(128, 16, 4, 16, torch.float16), (64, 6, 2, 32, torch.bfloat16)])
def test_prompts_decodes_and_extends(D, Hq, H, bs, dtype):
    pytest.importorskip("vllm")
    impl = B.TurboQuantB200EightBitImpl(Hq, D, 1 / math.sqrt(D), H)
    g = torch.Generator(device=DEV).manual_seed(5)
    blocks, n = 64, 3
    cache = torch.zeros(B.TurboQuantB200EightBitBackend.get_kv_cache_shape(blocks, bs, H, D), dtype=torch.uint8, device=DEV)
    tables = torch.randperm(blocks, generator=g, device=DEV)[:n * 20].view(n, 20).to(torch.int32)
    layer, lens = SimpleNamespace(layer_name="model.layers.0.self_attn.attn"), [0] * n
    K, V = [[] for _ in range(n)], [[] for _ in range(n)]
    for new in ((50, 7, 1), (1, 1, 1), (1, 40, 1), (33, 1, 150), (1, 1, 1)):
        T = sum(new)
        q, k, v = (torch.randn(T + 3, h * D, generator=g, device=DEV).to(dtype) for h in (Hq, H, H))
        lens = [a + b for a, b in zip(lens, new)]
        start = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device=DEV)
        slots = torch.cat([tables[i].long()[(p := torch.arange(lens[i] - new[i], lens[i], device=DEV)) // bs] * bs + p % bs for i in range(n)])
        meta = SimpleNamespace(num_actual_tokens=T, max_query_len=max(new), query_start_loc=start, block_table=tables, max_seq_len=max(lens),
                               seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        impl.do_kv_cache_update(layer, k[:T].view(T, H, D), v[:T].view(T, H, D), cache, slots)
        out = torch.full((T + 3, Hq * D), 5.0, dtype=dtype, device=DEV)
        assert impl.forward(layer, q, k, v, cache, meta, output=out) is out
        assert (out[T:] == 5).all()                                         # rows of padding
        a = 0
        for i in range(n):
            K[i].append(k[a:a + new[i]].view(-1, H, D).float())
            V[i].append(v[a:a + new[i]].view(-1, H, D).float())
            kk, vv = (torch.cat(x).repeat_interleave(Hq // H, 1) for x in (K[i], V[i]))
            s = torch.einsum("jhd,khd->hjk", q[a:a + new[i]].view(-1, Hq, D).float(), kk) / math.sqrt(D)
            hidden = torch.arange(len(kk), device=DEV) > torch.arange(len(kk) - new[i], len(kk), device=DEV)[:, None]
            want = torch.einsum("hjk,khd->jhd", s.masked_fill(hidden, -math.inf).softmax(-1), vv)
            got = out[a:a + new[i]].view(-1, Hq, D).float()
            # e4m3 values are within 2^-4 of what was given, at random signs
            assert (got - want).norm() <= 0.08 * want.norm()
            a += new[i]
    assert _native.read_status(DEV) == 0


@pytest.mark.parametrize("new", [(0, 1, 1, 0, 1), (1, 0, 0, 0, 1), (0, 0, 0, 0, 1)])
def test_decode_steps_in_which_some_requests_bring_no_token(new):
    """A request without tokens does not move the rows behind it to other requests' contexts."""
    pytest.importorskip("vllm")
    D, Hq, H, bs, n = 128, 8, 2, 16, len(new)
    impl = B.TurboQuantB200EightBitImpl(Hq, D, 1 / math.sqrt(D), H)
    g = torch.Generator(device=DEV).manual_seed(9)
    cache = torch.zeros(B.TurboQuantB200EightBitBackend.get_kv_cache_shape(4 * n, bs, H, D), dtype=torch.uint8, device=DEV)
    tables = torch.randperm(4 * n, generator=g, device=DEV).view(n, 4).to(torch.int32)
    lens = [33, 20, 64, 7, 50]
    layer = SimpleNamespace(layer_name="model.layers.0.self_attn.attn")
    for i in range(n):
        k, v = (torch.randn(lens[i], H, D, generator=g, device=DEV).half() for _ in range(2))
        p = torch.arange(lens[i], device=DEV)
        impl.do_kv_cache_update(layer, k, v, cache, tables[i].long()[p // bs] * bs + p % bs)
    T = sum(new)
    q = torch.randn(T, Hq * D, generator=g, device=DEV).half()
    step = lambda rows, which, starts: SimpleNamespace(
        num_actual_tokens=rows, max_query_len=1, query_start_loc=torch.tensor(starts, dtype=torch.int32, device=DEV), block_table=tables[which],
        seq_lens=torch.tensor([lens[i] for i in which], dtype=torch.int32, device=DEV), max_seq_len=64)
    starts = [0] + list(torch.tensor(new).cumsum(0))
    out = impl.forward(layer, q, None, None, cache, step(T, list(range(n)), starts), output=torch.full_like(q, 5.0))
    there = [i for i in range(n) if new[i]]
    want = impl.forward(layer, q, None, None, cache, step(T, there, list(range(T + 1))), output=torch.full_like(q, 5.0))
    assert torch.equal(out, want) and _native.read_status(DEV) == 0
