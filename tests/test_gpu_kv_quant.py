"""8-bit KV pages: codes and scales bit for bit the definition in float32, and
rows read back; slots, strides, page sizes, odd sizes, zeros, infinities, NaN."""
import numpy as np
import pytest

import vspec_b200 as V
from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

KINDS = {"fp8": V.KV_FP8, "int8": V.KV_INT8}
DTYPES = {"f32": V.T_F32, "f16": V.T_F16, "bf16": V.T_BF16}


def _torch_type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _definition(torch, x, kind):
    """Codes (bytes) and scales of rows [..., d], float32 arithmetic on the CPU."""
    x = x.float().cpu().numpy()
    most = np.float32(448 if kind == "fp8" else 127)
    with np.errstate(all="ignore"):
        top = np.where(np.isfinite(x), np.abs(x), np.float32(0)).max(-1)
        c = x * (most / top)[..., None]
        c = np.clip(np.where(np.isnan(c), np.float32(0), c), -most, most)
    if kind == "int8":
        return np.rint(c).astype(np.int8).view(np.uint8), top / most
    return torch.from_numpy(c).to(torch.float8_e4m3fn).view(torch.uint8).numpy(), top / most


def _append(torch, k, v, slots, pool, kind, name, stride=0):
    rows, heads, d = k.shape
    out = []
    for _ in range(2):
        out.append(torch.full((pool, heads, d), 0xA5, dtype=torch.uint8, device="cuda"))
        out.append(torch.full((pool, heads), -7.0, device="cuda"))
    V.kv_quant_append(k.data_ptr(), v.data_ptr(), slots.data_ptr() if slots is not None else None, rows, heads, d,
                      pool, KINDS[kind], out[0].data_ptr(), out[2].data_ptr(), out[1].data_ptr(), out[3].data_ptr(),
                      src_dtype=DTYPES[name], k_stride=stride, v_stride=stride)
    torch.cuda.synchronize()
    return out


def _check(torch, x, codes, scales, slots, kind):
    want_c, want_s = _definition(torch, x, kind)
    got_c, got_s = codes.cpu().numpy(), scales.cpu().numpy()
    at = np.arange(len(x)) if slots is None else slots.cpu().numpy()
    keep = (at >= 0) & (at < len(got_c))
    assert np.array_equal(got_s[at[keep]].view(np.uint32), want_s[keep].view(np.uint32))
    if kind == "fp8":   # the sign of a zero code is free
        same = (got_c[at[keep]] == want_c[keep]) | ((got_c[at[keep]] & 0x7F == 0) & (want_c[keep] & 0x7F == 0))
        assert same.all()
    else:
        assert np.array_equal(got_c[at[keep]], want_c[keep])
    rest = np.setdiff1d(np.arange(len(got_c)), at[keep])
    assert (got_c[rest] == 0xA5).all() and (got_s[rest] == -7.0).all()


def _rows(torch, rng, rows, heads, d, name):
    x = rng.standard_normal((rows, heads, d)).astype(np.float32) * np.exp(rng.uniform(-8, 8, (rows, heads, 1))).astype(np.float32)
    x[0, 0] = 0.0
    x[1 % rows, 0] = 1e-40
    x[2 % rows, -1, :2] = [np.inf, -np.inf][:d][:2] if d > 1 else np.inf
    x[3 % rows, 0, 0] = np.nan
    x[4 % rows, 0] = np.nan
    x[5 % rows, 0] = np.linspace(-63.5, 63.5, d)      # ties of int8 codes among them
    x[6 % rows, 0, 0] = 3e38
    return torch.from_numpy(x).to(_torch_type(torch, name)).cuda()


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256, 512, 80, 24, 33, 1])
def test_append_matches_definition(kind, name, d):
    torch = torch_cuda()
    rng = np.random.default_rng(d + len(name))
    for rows, heads in ((1, 1), (9, 3), (70, 8)):
        k, v = _rows(torch, rng, rows, heads, d, name), _rows(torch, rng, rows, heads, d, name)
        pool = rows + 13
        slots = torch.from_numpy(rng.permutation(pool)[:rows].astype(np.int32)).cuda()
        if rows > 8:
            slots[7] = -1                                 # a skipped row
        kc, ks, vc, vs = _append(torch, k, v, slots, pool, kind, name)
        _check(torch, k, kc, ks, slots, kind)
        _check(torch, v, vc, vs, slots, kind)
    assert V.page_fault_flag() == 0


@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_append_strides_and_bad_slots(kind):
    torch = torch_cuda()
    rng = np.random.default_rng(8)
    rows, heads, d = 21, 2, 64
    for extra in (0, 8, 3):                               # 3: rows that are not 16-byte aligned
        stride = 2 * heads * d + extra
        buf = torch.from_numpy(rng.standard_normal((rows, stride)).astype(np.float32)).cuda()
        k = buf[:, :heads * d].as_strided((rows, heads, d), (stride, d, 1))
        v = buf[:, heads * d:].as_strided((rows, heads, d), (stride, d, 1), heads * d)
        kc, ks, vc, vs = _append(torch, k, v, None, rows, kind, "f32", stride)
        _check(torch, k, kc, ks, None, kind)
        _check(torch, v, vc, vs, None, kind)
    V.page_fault_flag()
    k = torch.randn((3, heads, d), device="cuda")
    slots = torch.tensor([4, 5, 1], dtype=torch.int32, device="cuda")   # 5 is past the pool
    kc, ks, vc, vs = _append(torch, k, k, slots, 5, kind, "f32")
    assert V.page_fault_flag() == 1
    _check(torch, k, kc, ks, slots, kind)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,d,pt", [(8, 128, 16), (1, 64, 5), (3, 20, 1), (2, 33, 7), (5, 256, 64)])
def test_gather_reads_back_in_token_order(kind, name, heads, d, pt):
    torch = torch_cuda()
    rng = np.random.default_rng(heads * d + pt)
    lens = [0, 37, 1, 0, 64, 100, 0]
    need = [-(-n // pt) for n in lens]
    pages = sum(need) + 4
    perm = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lens), max(need) + 1), -1, dtype=np.int32)      # unused entries are never read
    o = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[o:o + n]
        o += n
    x = torch.from_numpy(rng.standard_normal((2, pages * pt, heads, d)).astype(np.float32)).cuda()
    kc, ks, vc, vs = _append(torch, x[0], x[1], None, pages * pt, kind, "f32")
    total = sum(lens)
    dt = _torch_type(torch, name)
    ko = torch.full((total + 2, heads, d), 3.0, dtype=dt, device="cuda")
    vo = torch.full((total + 2, heads, d), 3.0, dtype=dt, device="cuda")
    tab = torch.from_numpy(table).cuda()
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
    V.kv_quant_gather(kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), tab.data_ptr(), cu.data_ptr(),
                      len(lens), total + 2, heads, d, pt, table.shape[1], pages, KINDS[kind], ko.data_ptr(),
                      vo.data_ptr(), out_dtype=DTYPES[name])
    torch.cuda.synchronize()
    assert V.page_fault_flag() == 0
    rows = np.concatenate([table[b, np.arange(n) // pt].astype(np.int64) * pt + np.arange(n) % pt
                           for b, n in enumerate(lens) if n])
    at = torch.from_numpy(rows).cuda()
    for c, s, out in ((kc, ks, ko), (vc, vs, vo)):
        value = c.view(torch.int8).float() if kind == "int8" else c.view(torch.float8_e4m3fn).float()
        want = (value[at] * s[at].unsqueeze(-1)).to(dt)
        assert torch.equal(out[:total], want)
        assert (out[total:] == 3.0).all()                 # rows past the last sequence are left alone


def test_gather_bad_page_raises_the_flag():
    torch = torch_cuda()
    c = torch.zeros((4, 1, 16), dtype=torch.uint8, device="cuda")
    s = torch.ones((4, 1), device="cuda")
    out = torch.empty((4, 1, 16), device="cuda")
    tab = torch.tensor([[0, 9]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    V.page_fault_flag()
    V.kv_quant_gather(c.data_ptr(), c.data_ptr(), s.data_ptr(), s.data_ptr(), tab.data_ptr(), cu.data_ptr(), 1, 4, 1,
                      16, 2, 2, 2, V.KV_INT8, out.data_ptr(), out.data_ptr(), out_dtype=V.T_F32)
    torch.cuda.synchronize()
    assert V.page_fault_flag() == 1


def test_pool_offsets_past_32_bits():
    torch = torch_cuda()
    heads, d, pt = 8, 128, 16
    pool = (1 << 32) // (heads * d) + 64                  # codes pass 4 GiB
    kc = torch.empty((pool, heads, d), dtype=torch.uint8, device="cuda")
    ks = torch.empty((pool, heads), device="cuda")
    x = torch.randn((5, heads, d), device="cuda")
    y = torch.randn((5, heads, d), device="cuda")
    # K and V share the buffers: V's rows go to other slots by a second call
    last = pool // pt - 1
    slots = torch.tensor([last * pt + i for i in (0, 3, 5, 7, 15)], dtype=torch.int32, device="cuda")
    V.kv_quant_append(x.data_ptr(), x.data_ptr(), slots.data_ptr(), 5, heads, d, pool, V.KV_INT8, kc.data_ptr(),
                      kc.data_ptr(), ks.data_ptr(), ks.data_ptr())
    tab = torch.tensor([[last]], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, pt], dtype=torch.int32, device="cuda")
    out = torch.empty((2, pt, heads, d), device="cuda")
    V.kv_quant_gather(kc.data_ptr(), kc.data_ptr(), ks.data_ptr(), ks.data_ptr(), tab.data_ptr(), cu.data_ptr(), 1, pt,
                      heads, d, pt, 1, pool // pt, V.KV_INT8, out[0].data_ptr(), out[1].data_ptr(), out_dtype=V.T_F32)
    torch.cuda.synchronize()
    c, s = _definition(torch, x, "int8")
    want = c.view(np.int8).astype(np.float32) * s[..., None]
    assert np.array_equal(out[0].cpu().numpy()[[0, 3, 5, 7, 15]], want)
    assert V.page_fault_flag() == 0
    del y
