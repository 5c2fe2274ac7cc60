"""Refusals and host-side state of the paged 8-bit KV cache (CPU only, no kernel runs)."""

import pytest

torch = pytest.importorskip("torch")

from sparknet import _native, ops  # noqa: E402

pytestmark = pytest.mark.skipif(not _native.available(), reason="the extension is not built")

BF16 = torch.bfloat16


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def cache(pages=4, heads=2, page=16, dim=64):
    return ops.Fp8KVCache(pages, heads, page_size=page, head_dim=dim, device="cpu")


def rows(n=3, heads=2, dim=64, dtype=BF16):
    return torch.zeros(n, heads, dim, dtype=dtype)


def test_cache_state():
    c = cache()
    assert c.k.shape == c.v.shape == (4, 2, 16, 64) and c.k.dtype == torch.float8_e4m3fn
    assert c.k_scale.shape == c.v_scale.shape == (4, 2)
    assert c.nbytes() == 2 * 4 * 2 * (16 * 64 + 4)
    assert (c.num_pages, c.kv_heads, c.page_size, c.head_dim) == (4, 2, 16, 64)
    d = ops.Fp8KVCache.from_tensors(c.k, c.v, c.k_scale, c.v_scale)
    assert d.k.data_ptr() == c.k.data_ptr()


@pytest.mark.parametrize("kwargs", [{"page_size": 24}, {"page_size": 256}, {"head_dim": 96}, {"head_dim": 256},
                                    {"num_pages": 0}, {"kv_heads": 0}])
def test_cache_shapes_refused(kwargs):
    with pytest.raises(ValueError):
        ops.Fp8KVCache(**{"num_pages": 4, "kv_heads": 2, "device": "cpu", **kwargs})


def test_cache_tensors_refused():
    c = cache()
    for bad in ((c.k[:3], c.v, c.k_scale, c.v_scale), (c.k.view(torch.uint8), c.v, c.k_scale, c.v_scale),
                (c.k.transpose(1, 2), c.v.transpose(1, 2), c.k_scale, c.v_scale),
                (c.k, c.v, c.k_scale.double(), c.v_scale), (c.k, c.v, c.k_scale, c.v_scale[:2]),
                (c.k, c.v, c.k_scale[:, :1].expand(4, 2), c.v_scale)):
        with pytest.raises(ValueError):
            ops.Fp8KVCache.from_tensors(*bad)


@pytest.mark.parametrize("k,v,slots,word", [
    (rows(heads=1), rows(heads=1), i32(3), "rows must be"),
    (rows(), rows(n=2), i32(3), "rows must be"),
    (rows(dim=128), rows(dim=128), i32(3), "rows must be"),
    (rows(dtype=torch.float32), rows(dtype=torch.float32), i32(3), "bfloat16"),
    (rows(), rows(dtype=torch.float16), i32(3), "bfloat16"),
    (rows(dim=65)[..., :64], rows(), i32(3), "strides"),
    (rows(dim=128)[..., ::2], rows(), i32(3), "contiguous rows"),
    (rows(dim=72)[..., 4:68], rows(), i32(3), "16-byte"),
    (rows(), rows(), i32(4), "slots"),
    (rows(), rows(), i32(3).long(), "slots"),
    (rows(), rows(), i32(3, 1), "slots"),
    (rows(), rows(), i32(6)[::2], "slots"),
    (rows(), rows(), i32(3), "not on a CUDA device"),
])
def test_append_refused(k, v, slots, word):
    with pytest.raises(ValueError, match=word):
        ops.kv_append(cache(), k, v, slots)


@pytest.mark.parametrize("qkv,cos,positions,slots,q_out,word", [
    (torch.zeros(3, 4 * 64, dtype=BF16), torch.zeros(9, 32), i32(3), i32(3), None, "qkv"),
    (torch.zeros(3, 6 * 64 + 8, dtype=BF16), torch.zeros(9, 32), i32(3), i32(3), None, "qkv"),
    (torch.zeros(3, 6 * 64), torch.zeros(9, 32), i32(3), i32(3), None, "bfloat16"),
    (torch.zeros(3, 6 * 64, dtype=BF16), torch.zeros(9, 64), i32(3), i32(3), None, "cos and sin"),
    (torch.zeros(3, 6 * 64, dtype=BF16), torch.zeros(0, 32), i32(3), i32(3), None, "cos and sin"),
    (torch.zeros(3, 6 * 64, dtype=BF16), torch.zeros(9, 32).double(), i32(3), i32(3), None, "cos and sin"),
    (torch.zeros(3, 6 * 64, dtype=BF16), torch.zeros(9, 32), i32(2), i32(3), None, "positions"),
    (torch.zeros(3, 6 * 64, dtype=BF16), torch.zeros(9, 32), i32(3), i32(2), None, "slots"),
    (torch.zeros(3, 6 * 64, dtype=BF16), torch.zeros(9, 32), i32(3), i32(3), rows(heads=1), "q_out"),
    (torch.zeros(3, 6 * 64, dtype=BF16), torch.zeros(9, 32), i32(3), i32(3), rows(dtype=torch.float16), "q_out"),
    (torch.zeros(3, 6 * 64, dtype=BF16), torch.zeros(9, 32), i32(3), i32(3), None, "not on a CUDA device"),
])
def test_rope_append_refused(qkv, cos, positions, slots, q_out, word):
    with pytest.raises(ValueError, match=word):
        ops.rope_kv_append(cache(), qkv, cos, cos, positions, slots, q_out)


def test_read_refused():
    c = cache()
    for slots, kwargs, word in ((i32(3).long(), {}, "slots"), (i32(3, 2), {}, "slots"),
                                (i32(3), {"dtype": torch.float64}, "dtype"),
                                (i32(3), {"k_out": rows(n=2)}, "k_out"),
                                (i32(3), {"v_out": rows(dtype=torch.float16)}, "v_out"),
                                (i32(3), {}, "not on a CUDA device")):
        with pytest.raises(ValueError, match=word):
            ops.kv_read(c, slots, **kwargs)


def q(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("query,tables,lengths,kwargs,word", [
    (q(2, 64), i32(2, 3), i32(2), {}, "q must be"),
    (q(2, 4, 128), i32(2, 3), i32(2), {}, "head_dim"),
    (q(2, 3, 64), i32(2, 3), i32(2), {}, "multiple of the cache's"),
    (q(2, 0, 64), i32(2, 3), i32(2), {}, "multiple of the cache's"),
    (q(2, 4, 64, dtype=torch.float32), i32(2, 3), i32(2), {}, "bfloat16"),
    (q(2, 0, 4, 64), i32(2, 3), i32(2), {}, "query rows"),
    (q(2, 4, 65)[..., :64], i32(2, 3), i32(2), {}, "strides"),
    (q(2, 4, 72)[..., 4:68], i32(2, 3), i32(2), {}, "16-byte"),
    (q(2, 4, 64), i32(3, 3), i32(2), {}, "block_tables"),
    (q(2, 4, 64), i32(2, 0), i32(2), {}, "block_tables"),
    (q(2, 4, 64), i32(2, 3).long(), i32(2), {}, "block_tables"),
    (q(2, 4, 64), i32(3, 2).t(), i32(2), {}, "block_tables"),
    (q(2, 4, 64), i32(2, 3), i32(3), {}, "lengths"),
    (q(2, 4, 64), i32(2, 3), i32(2).long(), {}, "lengths"),
    (q(2, 4, 64), i32(2, 3), i32(2), {"window": -1}, "window"),
    (q(2, 4, 64), i32(2, 3), i32(2), {"scale": float("inf")}, "scale"),
    (q(2, 4, 64), i32(2, 3), i32(2), {"out": q(2, 4, 64, dtype=torch.float16)}, "out"),
    (q(2, 4, 64), i32(2, 3), i32(2), {"out": q(2, 64, 4).transpose(1, 2)}, "out"),
    (q(2, 4, 64), i32(2, 3), i32(2), {}, "not on a CUDA device"),
])
def test_attention_refused(query, tables, lengths, kwargs, word):
    with pytest.raises(ValueError, match=word):
        ops.paged_decode_attention(query, cache(), tables, lengths, **kwargs)


@pytest.mark.parametrize("change,word", [
    ({"lengths": i32(2).long()}, "lengths"),
    ({"new_tokens": i32(3)}, "new_tokens"),
    ({"block_tables": i32(2, 0)}, "block_tables"),
    ({"block_tables": i32(4, 2).t()}, "block_tables"),
    ({"free_pages": i32(8)[::2]}, "free_pages"),
    ({"free_count": i32(2)}, "free_count"),
    ({"page_size": 48}, "page_size"),
    ({"max_tokens": -1}, "max_tokens"),
    ({"max_tokens": 1 << 30}, "max_tokens"),
    ({"finished": i32(2)}, "finished"),
    ({"lengths_out": i32(1)}, "lengths_out"),
    ({"free_count_out": i32(0)}, "free_count_out"),
    ({"lengths": i32(0), "new_tokens": i32(0), "block_tables": i32(0, 4)}, "4096 requests"),
    ({"lengths": i32(4097), "new_tokens": i32(4097), "block_tables": i32(4097, 4)}, "4096 requests"),
    ({}, "not on a CUDA device"),
])
def test_plan_refused(change, word):
    args = {"lengths": i32(2), "new_tokens": i32(2), "block_tables": i32(2, 4), "free_pages": i32(8),
            "free_count": i32(1), "page_size": 16, "max_tokens": 8} | change
    with pytest.raises(ValueError, match=word):
        ops.plan_pages(args.pop("lengths"), args.pop("new_tokens"), args.pop("block_tables"), args.pop("free_pages"),
                       args.pop("free_count"), **args)


def test_page_table_state():
    t = ops.PageTable(6, page_size=16, max_requests=2, max_pages=4, device="cpu")
    assert t.free_pages.tolist() == [5, 4, 3, 2, 1, 0] and t.free_count.tolist() == [6]
    assert t.block_tables.shape == (2, 4) and t.lengths.tolist() == [0, 0]
    for bad in ({"num_pages": 0}, {"max_requests": 0}, {"max_pages": 0}):
        with pytest.raises(ValueError):
            ops.PageTable(**{"num_pages": 6, "page_size": 16, "max_requests": 2, "max_pages": 4, "device": "cpu",
                             **bad})


@pytest.mark.parametrize("slots,fine", [
    ([31, 64, 33 + 64 * 2, 127, 5], False),        # 31 and 5 share page 0
    ([31, 64, 33 + 64 * 2, 127], True),
    ([30, 31, 32, 33], True),                      # one sequence over a page's end
    ([32, 33, 35], False),
    ([33, 33], False),                             # the same slot twice
    ([0, -1, 1], False),                           # a skipped row ends a run
    ([-1, 1 << 30, -1, 7], True),
])
def test_append_checks_slots(slots, fine):
    """check=True refuses two runs for one page before anything is launched."""
    c = cache(pages=6, page=32)
    at = torch.tensor(slots, dtype=torch.int32)
    n = len(slots)
    word = "not on a CUDA device" if fine else "two separate runs"
    with pytest.raises(ValueError, match=word):
        ops.kv_append(c, rows(n), rows(n), at, check=True)
    with pytest.raises(ValueError, match=word):
        ops.rope_kv_append(c, torch.zeros(n, 6 * 64, dtype=BF16), torch.zeros(9, 32), torch.zeros(9, 32), i32(n), at,
                           check=True)
