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


def test_tensors():
    """Tensors that the device could not read, or that end too early, are refused before a call."""
    torch = pytest.importorskip("torch")
    i32 = torch.zeros(8, dtype=torch.int32)
    for args in [(i32, 16, 16), (16, i32, 16), (16, 16, i32)]:  # (host memory)
        with pytest.raises(TypeError):
            ha.KVBatch(2, 2, 1, 1, *args, 4)
    assert ha.KVBatch(2, 2, 1, 1, 16, 32, 48, 4).c.table_stride == 4
    with pytest.raises(ValueError):
        ha.PagedKV(torch.zeros(1 << 20, dtype=torch.uint8), 4)


@pytest.mark.gpu
def test_device_tensors():
    torch = pytest.importorskip("torch")
    ok = [torch.zeros(n, dtype=torch.int32, device="cuda:0") for n in (3, 2, 8)]
    ha.KVBatch(2, 2, 1, 1, *ok, 4)
    for k in range(3):
        for x in (ok[k][:-1], ok[k].long(), ok[k].cpu(), torch.zeros(32, dtype=torch.int32, device="cuda:0")[::2]):
            with pytest.raises(TypeError):
                ha.KVBatch(2, 2, 1, 1, *[x if j == k else ok[j] for j in range(3)], 4)
    nb = ha.PagedKV.page_bytes()
    pool = torch.zeros(3 * nb + 16, dtype=torch.uint8, device="cuda:0")
    ha.PagedKV(pool, 3).close()
    for bad in (pool[:3 * nb - 1], pool.cpu()):
        with pytest.raises(ValueError):
            ha.PagedKV(bad, 3)
    with pytest.raises(ValueError):
        ha.PagedKV(pool, 2, n_layers=2)
