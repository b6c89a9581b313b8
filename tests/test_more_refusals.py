"""What the serving step's newer calls refuse, they refuse before anything of the device is touched (no GPU: the context is a stand-in that nothing looks into)."""
import ctypes as C
from types import SimpleNamespace

import pytest

import recipe_dev_b200 as rq
from recipe_dev_b200 import capi


@pytest.fixture(scope="module")
def lib():
    return rq.load_library()


def refused(lib, status, why):
    assert status < 0
    text = lib.rq_last_error().decode()
    assert why in text, text


CTX = C.cast(C.create_string_buffer(1 << 16), C.c_void_p)
AT = 4096  # an address that nothing reads


@pytest.mark.parametrize("change,why", [(dict(ctx=None), "null"), (dict(logits=0), "null"), (dict(token=0), "null"), (dict(rows=0), "positive"), (dict(vocabulary=0), "positive"), (dict(stride=99), "row_stride"),
                                        (dict(vocabulary=1048577, stride=1048577), "at most 1048576"), (dict(rows=(1 << 26) + 1), "2^26"), (dict(top=-1), "from 0 to 64"), (dict(top=65), "from 0 to 64"),
                                        (dict(top=3, top_token=0, top_logprob=0), "alternatives"), (dict(logits=AT + 2), "aligned")])
def test_logprobs(lib, change, why):
    a = dict(ctx=CTX, logits=AT, stride=100, rows=4, vocabulary=100, token=AT, logprob=AT, entropy=AT, rank=AT, top=3, top_token=AT, top_logprob=AT, stream=None) | change
    refused(lib, lib.rq_logprobs(*a.values()), why)


@pytest.mark.parametrize("change,why", [(dict(ctx=None), "null"), (dict(x=0), "null"), (dict(delta=0), "null"), (dict(out=0), "null"), (dict(y=0), "null"), (dict(n=0), "positive"), (dict(tokens=0), "positive"),
                                        (dict(n=1 << 32), "2^31"), (dict(xs=63), "at least n"), (dict(ds=63), "at least n"), (dict(os=0), "at least n"), (dict(ys=-64), "at least n"),
                                        (dict(gate=AT, gk=2), "gate_k_stride"), (dict(gate=AT, gt=-1), "gate_t_stride"), (dict(epsilon=-1e-6), "epsilon"), (dict(epsilon=float("nan")), "epsilon")])
def test_residual_norm(lib, change, why):
    a = dict(ctx=CTX, x=AT, xs=64, delta=AT, ds=64, n=64, tokens=2, delta_gain=0, gate=0, gk=0, gt=0, scale=1.0, gain=0, epsilon=1e-6, out=AT, os=64, y=AT, ys=64, stream=None) | change
    refused(lib, lib.rq_residual_norm(*a.values()), why)


CACHE = dict(k=AT, v=AT, type=capi.KV_INT8, heads=2, head_dim=128, page_size=16, pages=4, page_stride=4096, head_stride=2048, line_stride=128, k_scale=AT, v_scale=AT, scale_page=32, scale_head=16,
             scale_line=1)


@pytest.mark.parametrize("change,why", [(dict(type=3), "INT8(2)"), (dict(type=-1), "INT8(2)"), (dict(k_scale=0), "k_scale"), (dict(v_scale=0), "v_scale"), (dict(v_scale=AT + 2), "aligned"), (dict(k=AT + 8), "16-byte"),
                                        (dict(line_stride=136), "multiples of 16"), (dict(page_stride=4104), "multiples of 16"), (dict(head_stride=24), "multiples of 16"), (dict(scale_page=-1), "not be negative"),
                                        (dict(scale_line=1 << 31), "2^31"), (dict(head_dim=96), "64, 128 or 256"), (dict(page_size=12), "power of two"), (dict(pages=1 << 27), "2^31")])
@pytest.mark.parametrize("call", ["store", "attention"])
def test_caches(lib, change, why, call):
    cache = capi._KvCacheStruct(*(CACHE | change).values())
    at = C.addressof(cache)
    if call == "store":
        status = lib.rq_rope_store(CTX, AT, 512, 4, AT, 256, AT, 256, 3, 0, 0, 1e-6, 0, 0, 0, 0, AT, AT, AT, 512, at, None)
    else:
        status = lib.rq_attention(CTX, AT, 512, 4, at, AT, 8, 8, AT, AT, 2, 3, 1, 0.1, 0, AT, 512, None)
    refused(lib, status, why)


def test_a_cache_of_16_bits_asks_for_no_scales(lib):
    """What lies behind the fields that such a cache has is not looked at (a host's older structure ends there)."""
    cache = capi._KvCacheStruct(*(CACHE | dict(type=capi.KV_F16, k_scale=1, v_scale=3, scale_page=-5)).values())
    refused(lib, lib.rq_attention(CTX, AT, 512, 4, C.addressof(cache), AT, 8, 8, AT, AT, 2, 3, 1, -1.0, 0, AT, 512, None), "scale must be finite")


def test_tensors_of_the_wrong_place():
    torch = pytest.importorskip("torch")
    codes, scales = torch.zeros((2, 2, 16, 64), dtype=torch.int8), torch.zeros((2, 2, 16))
    with pytest.raises(ValueError, match="CUDA"):
        rq.KvCache(codes, codes, scales, scales)
    ctx = rq.Context.__new__(rq.Context)  # (a device's context that was never made)
    ctx.lib, ctx.handle, ctx.device = rq.load_library(), 0, 0
    plane, ints = torch.zeros((2, 64)), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device"):
        ctx.logprobs(plane, ints)
    with pytest.raises(ValueError, match="device"):
        ctx.residual_norm(plane, plane)


def test_the_small_decoder():
    pytest.importorskip("torch")
    from recipe_dev_b200 import serve

    for how in (dict(norms="behind"), dict(residual_scale=0.5)):
        with pytest.raises(ValueError, match="norms"):
            serve.Decoder(None, 1, 64, 1, 1, 64, 64, 10, 4, **how)
    for n in (-1, 65):
        with pytest.raises(ValueError, match="alternatives"):
            serve.Batch(SimpleNamespace(positions=32, vocabulary=100), [[1]], 1, logprobs=n)
