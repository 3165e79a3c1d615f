"""Page clears of more pages than one launch's grid holds, and the session creation that
asks for them."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
MANY = 65535 + 40


def _nova():
    import nova_amd
    return nova_amd.load("qwen25_1p5b")


def _pages(last):
    """pages 1 and 2 again and again, then one more"""
    pages = 1 + np.arange(MANY, dtype=np.int32) % 2
    pages[-1] = last
    return pages


def test_q8_clears():
    nova, nb = _nova(), 6
    host = np.random.default_rng(1).integers(0, 256, (nova.n_layers, nb, nova.kv_q8_page_bytes()), dtype=np.uint8)
    dev, dp = nova.upload(host), nova.upload(_pages(4))
    nova.launch_kv_q8_zero_pages(dev.ptr, nb, dp.ptr, MANY, None)
    nova.dev_sync()
    host[:, [1, 2, 4]] = 0
    assert np.array_equal(dev.numpy(host.shape, np.uint8), host)


def test_fp16_clears():
    nova, nb = _nova(), 6
    shape = (nova.n_layers, nb, nova.kb * nova.kvw)
    hosts = [np.random.default_rng(s).integers(1, 60000, shape).astype(np.uint16) for s in (2, 3)]
    k, v = (nova.upload(h) for h in hosts)
    dp = nova.upload(_pages(4))
    nova.launch_kv_zero_pages(k.ptr, v.ptr, nb, dp.ptr, MANY, None)
    nova.dev_sync()
    for dev, host in zip((k, v), hosts):
        host[:, [1, 2, 4]] = 0
        assert np.array_equal(dev.numpy(shape, np.uint16), host)


def test_sessions_of_more_pages():
    """128 sessions of 8192 tokens and one more, 66048 8-bit pages"""
    nova, n = _nova(), 129
    h = nova.nova_paged_new_q8(n, 8192)
    nb, page = nova.nova_paged_nb(h), nova.kv_q8_page_bytes()
    assert nb > 65535
    pool = nova.nova_paged_pool_q8(h)
    noise = np.full(page, 0x5a, np.uint8)
    at = [(layer * nb + p) * page for layer in (0, nova.n_layers - 1) for p in (0, 65534, 65535, nb - 1)]
    for off in at:
        nova.dev_upload(pool + off, noise.ctypes.data, page)
    ids = (C.c_int * n)()
    assert nova.nova_paged_create_sessions(h, n, 1, ids) == n
    for off in at:
        assert not nova.download(pool, (page,), np.uint8, off).any()
    nova.nova_paged_delete(h)
