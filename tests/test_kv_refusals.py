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


class Fake:
    """A tensor's attributes, without memory."""

    def __init__(self, n, dtype="float16", gpu=0, contiguous=True, cuda=True):
        self.n, self.dtype, self.is_cuda, self.contiguous = n, "torch." + dtype, cuda, contiguous
        self.device = type("Device", (), {"index": gpu if cuda else None})

    def data_ptr(self):
        return 4096

    def numel(self):
        return self.n

    def is_contiguous(self):
        return self.contiguous

    def element_size(self):
        return 4 if "32" in self.dtype else 2

    def untyped_storage(self):
        n = self.n * self.element_size()
        return type("Storage", (), {"nbytes": staticmethod(lambda: n)})

    def storage_offset(self):
        return 0

    def stride(self, dim):
        return 1 if self.contiguous else 2


@pytest.mark.parametrize("dtype,f32", [(ha.F16, False), (ha.F32, True)])
def test_tensors_of_a_call(dtype, f32):
    """rows, q, values and out that the device could not read or write, or that end too early, and a batch of another GPU."""
    ha.load_library()
    kv = object.__new__(ha.PagedKV)
    kv._h = None  # (a call that gets past the checks has an invalid handle)
    kv.cfg = ha.HaKvConfig(1, 4, 16, 100, 4, 2, 128, 0, 1, dtype, 1e4, 1e-6, 0.0)
    kv._sizes(1)
    rt, width = "float32" if f32 else "float16", 4 * 2 * 128 + 2 * 2 * 128
    stride, nq, nv = width + 64, 3 * 4 * 128, 3 * 2 * 2 * 128
    nr = 2 * stride + width
    ints = [Fake(n, "int32", gpu=1) for n in (3, 2, 8)]
    b = ha.KVBatch(2, 3, 2, 20, *ints, 4)

    def append(rows=None, q=None, values=None, batch=b):
        kv.append(0, batch, rows or Fake(nr, rt, 1), stride, q or Fake(nq, gpu=1), values or Fake(nv, gpu=1))

    def attention(rows=None, q=None, out=None, batch=b):
        kv.attention(0, batch, q or Fake(nq, gpu=1), rows or Fake(nr, rt, 1), stride, out or Fake(nq, gpu=1))

    for call, args in ((append, {}), (append, dict(rows=4096, q=4096, values=4096)), (attention, {}), (attention, dict(rows=4096, q=4096, out=4096))):
        with pytest.raises(ha.HAError) as ei:
            call(**args)
        assert ei.value.code == ha.HA_ERR_HANDLE
    for call, names in ((append, dict(rows=nr, q=nq, values=nv)), (attention, dict(rows=nr, q=nq, out=nq))):
        for name, n in names.items():
            t = rt if name == "rows" else "float16"
            for bad in (Fake(n - 1, t, 1), Fake(n, "bfloat16", 1), Fake(n, "float16" if t == "float32" else "float32", 1), Fake(n, t, 0),
                        Fake(n, t, 1, contiguous=False), Fake(n, t, cuda=False)):
                with pytest.raises(TypeError):
                    call(**{name: bad})
        with pytest.raises(TypeError):
            call(batch=ha.KVBatch(2, 3, 2, 20, *[Fake(n, "int32", 0) for n in (3, 2, 8)], 4))
    for other in ([Fake(3, "int32", 0)] + ints[1:], ints[:2] + [Fake(8, "int32", 0)]):
        with pytest.raises(TypeError):
            ha.KVBatch(2, 3, 2, 20, *other, 4)


@pytest.mark.gpu
def test_device_tensors_of_a_call():
    torch = pytest.importorskip("torch")
    pool = torch.zeros(4 * ha.PagedKV.page_bytes(16, 2, 128), dtype=torch.uint8, device="cuda:0")
    kv = ha.PagedKV(pool, 4, page_size=16, max_ctx=64, HQ=4, HK=2, HD=128, rot_dim=0)
    up = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda:0")  # noqa: E731
    b = ha.KVBatch(2, 3, 2, 20, up(0, 2, 3), up(20, 5), up(0, 1, 2, 3), 2)
    width = 4 * 2 * 128 + 2 * 2 * 128
    wide = torch.randn(3, width + 64, device="cuda:0").half()
    q, out = (torch.zeros(3, 4, 128, dtype=torch.float16, device="cuda:0") for _ in "qo")
    values = torch.zeros(3, 2, 2, 128, dtype=torch.float16, device="cuda:0")
    kv.append(0, b, wide[:, :width], width + 64, q, values)  # (rows may lie apart; the last ends before the padding)
    kv.attention(0, b, q, wide, width + 64, out)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and (values != 0).any()
    for bad in (q[:2], q.float(), q.cpu(), q.transpose(0, 1)):
        with pytest.raises(TypeError):
            kv.append(0, b, wide, width + 64, bad)
        with pytest.raises(TypeError):
            kv.attention(0, b, bad, wide, width + 64, out)
        with pytest.raises(TypeError):
            kv.attention(0, b, q, wide, width + 64, bad)
    for bad in (wide[:2], wide.float(), wide.cpu(), wide[1:]):
        with pytest.raises(TypeError):
            kv.append(0, b, bad.contiguous() if len(bad) < 3 else bad, width + 64, q)
    with pytest.raises(TypeError):
        kv.append(0, b, wide, width + 64, q, values[:2])
    kv.close()
