"""Calls of the paged cache that are refused, and their neighbours that are not."""
import ctypes as C

import numpy as np
import pytest

from kestrel_amd.kmoe import F16, KmoeError, PagedKV
from tests.test_gpu_paged import _dev, ctx  # noqa: F401  (ctx: a fixture)

pytestmark = pytest.mark.gpu


def test_rotated_q_over_an_input(ctx):  # noqa: F811
    """q_out over any byte of q, k, v or the frequencies is refused, before anything is written; between them it is not."""
    import torch

    nh, nkv, hd, S = 4, 2, 64, 3
    kv, w, n = PagedKV(F16, nkv, hd, 32), nkv * hd, nh * hd
    pages = torch.zeros((4, kv.page_bytes), dtype=torch.uint8, device="cuda")
    b = ctx.paged_batch(_dev([[0, 1]] * 1, np.int32), _dev([40], np.int32), _dev([0, S], np.int32), S)
    size, stride = S * n, 2 * S * n  # rows far enough apart for q_out to lie between two of them
    buf = torch.ones(8 * stride, device="cuda")
    at = buf.data_ptr()
    inv = torch.ones(hd // 2, device="cuda")

    def call(q, k, v, out, qs=stride, ks=stride, vs=stride, fr=inv.data_ptr()):
        return ctx.lib.kmoe_paged_rope_kv_store(ctx.h, C.byref(kv.desc(pages)), pages.data_ptr(), C.byref(b), at + 4 * q, qs,
                                                at + 4 * k, ks, at + 4 * v, vs, nh, hd, fr, 1, at + 4 * out)

    q, k, v, far = 0, n, n + w, 6 * stride
    keep = buf.clone()
    for out in (q, q + 1, k, v, v + w - 1, stride - size + 1, stride, stride + n + 2 * w - 1, 2 * stride + n + 2 * w - 1):
        assert call(q, k, v, out) == -1, out
    for one in range(3):  # each of them alone
        a = [0, 0, 0]
        a[one] = far
        width = n if one == 0 else w
        for out in (far, far + width - 1, far + 1 - size):
            b1 = [x if i == one else 5 * stride - 8 * w for i, x in enumerate(a)]
            assert call(*b1, out, qs=n, ks=w, vs=w) == -1, (one, out)
    assert call(q, k, v, 4 * stride, fr=at + 4 * (4 * stride + size - 1)) == -1
    torch.cuda.synchronize()
    assert torch.equal(buf, keep) and not pages.any()
    for out in (n + 2 * w, stride - size, 2 * stride + n + 2 * w, 4 * stride):  # between two rows, and behind the last
        assert call(q, k, v, out) == 0, out
    torch.cuda.synchronize()
    same = torch.ones((S, n), device="cuda")
    with pytest.raises(KmoeError):
        ctx.paged_rope_kv_store(kv, pages, b, same, torch.ones((S, w), device="cuda"), torch.ones((S, w), device="cuda"), nh,
                                hd, inv, True, q_out=same)


def test_more_copies_than_pages(ctx):  # noqa: F811
    """Some page would be copied onto twice: refused before the arrays are read."""
    import torch

    kv = PagedKV(F16, 1, 64, 32)
    pages = torch.zeros((2, 4, kv.page_bytes), dtype=torch.uint8, device="cuda")
    one = np.zeros(1, np.int32)
    for n in (5, 2 ** 40, 2 ** 62, 2 ** 63 - 1):
        assert ctx.lib.kmoe_pages_copy(ctx.h, C.byref(kv.desc(pages, 2)), pages.data_ptr(), 2, pages.nbytes // 2,
                                       one.ctypes.data, one.ctypes.data, n) == -1


def test_page_numbers_past_32_bits(ctx):  # noqa: F811
    """Page numbers are not taken modulo 2^32."""
    import torch

    kv = PagedKV(F16, 1, 64, 32)
    pages = torch.arange(2 * 4 * kv.page_bytes, device="cuda").to(torch.uint8).view(2, 4, -1)
    pages[:, 1:] = 0
    keep = pages.clone()
    for s, d in ((np.array([2 ** 32]), np.array([1])), (np.array([0]), np.array([2 ** 32 + 1])), ([2 ** 32], [1]),
                 (torch.tensor([-2 ** 32]), [1])):
        with pytest.raises((ValueError, KmoeError)):
            ctx.pages_copy(kv, pages, s, d, n_layer=2)
    torch.cuda.synchronize()
    assert torch.equal(pages, keep)
    ctx.pages_copy(kv, pages, np.array([0], np.int64), torch.tensor([3]), n_layer=2)
    torch.cuda.synchronize()
    assert torch.equal(pages[:, 3], keep[:, 0])


def test_layers_of_whole_pages(ctx):  # noqa: F811
    """n_layer parts of a buffer whose parts are no whole pages: no layer begins where the copy would look for it."""
    import torch

    kv = PagedKV(F16, 1, 64, 32)
    pages = torch.zeros((3, 5, kv.page_bytes), dtype=torch.uint8, device="cuda")
    for n_layer in (2, 4, 0, -1):
        with pytest.raises(ValueError):
            ctx.pages_copy(kv, pages, [0], [1], n_layer=n_layer)
    ctx.pages_copy(kv, pages, [0], [4], n_layer=3)
    ctx.pages_copy(kv, pages, [0], [14], n_layer=1)
    torch.cuda.synchronize()
