"""What the paged 4-bit K/V cache refuses, on the CPU: configs, before any device is looked for, and handles."""
import ctypes

import pytest

import hybrid_attention as ha


@pytest.mark.parametrize("over,msg", [
    (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"), (dict(page_size=512), "page_size"),
    (dict(HD=64), "head_dim"), (dict(HD=192), "head_dim"), (dict(HQ=7), "multiple of HK"), (dict(HQ=34), "16 times HK"),
    (dict(HK=0), "multiple of HK"), (dict(HQ=2048, HK=128), "1024"), (dict(rot_dim=12), "rotary_dim"), (dict(rot_dim=264), "rotary_dim"),
    (dict(rot_dim=-8), "rotary_dim"), (dict(dtype=2), "dtype"), (dict(rope_theta=0.0), "rope_theta"),
    (dict(rope_theta=float("nan")), "rope_theta"), (dict(eps=0.0), "eps"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(n_pages=0), "n_pages"), (dict(n_layers=0), "n_layers"), (dict(max_ctx=0), "max_ctx"),
    (dict(max_ctx=(1 << 24) + 1), "max_ctx")])
def test_configs(over, msg):
    with pytest.raises(ha.HAError) as ei:
        ha.PagedKV(16, **{"n_pages": 4, **over})
    assert ei.value.code == ha.HA_ERR_ARG and msg in str(ei.value)


@pytest.mark.parametrize("pages", [None, 8])
def test_pages(pages):
    with pytest.raises(ha.HAError) as ei:
        ha.PagedKV(pages, 4)
    assert ei.value.code == ha.HA_ERR_ARG and "pages" in str(ei.value)


def test_no_device_is_a_device_error():
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(ha.HAError) as ei:
        ha.PagedKV(16, 4)
    assert ei.value.code == ha.HA_ERR_DEVICE


@pytest.mark.parametrize("page,HK,HD,want", [(64, 2, 256, 2 * 2 * 64 * 144), (16, 1, 128, 2 * 16 * 80), (256, 8, 256, 8 * 2 * 256 * 144)])
def test_page_bytes(page, HK, HD, want):
    assert ha.PagedKV.page_bytes(page, HK, HD) == want


def test_handles():
    lib = ha.load_library()
    buf = (ctypes.c_uint32 * 64)()
    buf[0] = 0x48414B56
    for h in (None, ctypes.cast(buf, ctypes.c_void_p)):
        assert lib.ha_kv_set_param(h, 0, b"q_norm", None, 256) == ha.HA_ERR_HANDLE
        assert lib.ha_kv_append(h, 0, None, None, 0, None, None, None) == ha.HA_ERR_HANDLE
        assert lib.ha_kv_attention(h, 0, None, None, None, 0, None, None) == ha.HA_ERR_HANDLE
        if h is not None:
            assert lib.ha_kv_destroy(h) == ha.HA_ERR_HANDLE
    assert lib.ha_kv_destroy(None) == ha.HA_OK
    assert lib.ha_kv_create(None, None, 0, None) == ha.HA_ERR_ARG
    assert lib.ha_kv_page_bytes(None, None) == ha.HA_ERR_ARG
    assert buf[0] == 0x48414B56
