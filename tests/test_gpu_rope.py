"""Rotary positions against the formula in 64 bits: layouts, part of the head,
scalings, types, strides, in place, long positions, and the inverse as the
gradient (against the adjoint identity and against differences)."""
import numpy as np
import pytest

import vspec_b200 as V
from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

DTYPES = {"f32": V.T_F32, "f16": V.T_F16, "bf16": V.T_BF16}


def _torch_type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _freqs64(rot, theta, scaling, factor, original, fast, slow):
    """f_i and the factor, from the definitions, in Python floats."""
    import math
    f, mult = [], 1.0
    if scaling == V.ROPE_NTK:
        theta = theta * factor ** (rot / (rot - 2)) if rot > 2 else theta * factor ** rot
    for i in range(rot // 2):
        x = theta ** (-2.0 * i / rot)
        if scaling == V.ROPE_LINEAR:
            x /= factor
        if scaling == V.ROPE_YARN:
            def pair(turns):
                return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
            lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
            ramp = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
            x = x * (1 - ramp) + x / factor * ramp
            mult = 0.1 * math.log(factor) + 1
        f.append(x)
    return np.array(f), mult


def _ref64(x, pos, turns, rot, inter, mult, sign=1.0):
    """x [t][h][d] float64 on the CPU; turns uint64 -> exact fraction of a turn."""
    frac = np.array([[(int(p) * int(f)) % (1 << 64) for f in turns] for p in pos], dtype=np.float64) / 2.0 ** 64
    ang = 2 * np.pi * frac
    c, s = (np.cos(ang) * mult)[:, None, :], (np.sin(ang) * mult * sign)[:, None, :]
    y = x.copy()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    ya, yb = a * c - b * s, a * s + b * c
    if inter:
        y[..., 0:rot:2], y[..., 1:rot:2] = ya, yb
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = ya, yb
    return y


# A coefficient is off by at most 2^-25 half turns of angle (9.4e-8), 2 ulp of sincospif (1.2e-7) and its
# product with the factor (6e-8); two products and a sum add 3 * 2^-24 of the terms: below 5e-7 of |a| + |b|.
# The result's own rounding is half an ulp of its type.
def _bound(x, y, rot, inter, mult, name):
    b = np.zeros_like(x)
    u, v = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    t = (np.abs(u) + np.abs(v)) * mult * 5e-7
    if inter:
        b[..., 0:rot:2], b[..., 1:rot:2] = t, t
    else:
        b[..., :rot // 2], b[..., rot // 2:rot] = t, t
    half_ulp = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[name]
    return b * (1 + half_ulp) + np.abs(y) * half_ulp + (2.0 ** -25 if name == "f16" else 1e-37)


def _call(torch, x_q, x_k, pos, turns, rot, name, inter, mult, inverse=False, q_out=None, k_out=None, **kw):
    t, hq, d = x_q.shape
    q_out = torch.empty_like(x_q, memory_format=torch.contiguous_format) if q_out is None else q_out
    hk = 0
    if x_k is not None:
        hk = x_k.shape[1]
        k_out = torch.empty_like(x_k, memory_format=torch.contiguous_format) if k_out is None else k_out
    V.rope(x_q.data_ptr(), x_k.data_ptr() if x_k is not None else None, q_out.data_ptr(),
           k_out.data_ptr() if x_k is not None else None, pos.data_ptr(), turns.data_ptr(), t, hq, hk, d, rot,
           DTYPES[name], interleaved=inter, inverse=inverse, attn_factor=mult, **kw)
    return q_out, k_out


def _turns_dev(torch, turns):
    return torch.from_numpy(turns.view(np.int64)).cuda()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (128, 64), (80, 20), (64, 16), (96, 36), (256, 256), (10, 6), (2, 2),
                                   (512, 510)])
def test_rope_matches_formula(name, inter, d, rot):
    torch = torch_cuda()
    rng = np.random.default_rng(d * 7 + rot + inter)
    dt = _torch_type(torch, name)
    turns, mult = V.rope_turns(rot, 1e6, V.ROPE_YARN, 4.0, 8192)
    for tokens, hq, hk in ((1, 1, 1), (5, 6, 2), (33, 3, 0)):
        q = torch.from_numpy(rng.standard_normal((tokens, hq, d))).to(dt).cuda()
        k = torch.from_numpy(rng.standard_normal((tokens, hk, d))).to(dt).cuda() if hk else None
        pos = rng.integers(0, 1 << 20, size=tokens).astype(np.int32)
        pos[0] = 0
        if tokens > 1:
            pos[1], pos[2] = (1 << 31) - 1, -3
        qo, ko = _call(torch, q, k, torch.from_numpy(pos).cuda(), _turns_dev(torch, turns), rot, name, inter, mult)
        torch.cuda.synchronize()
        for x, y in ((q, qo), (k, ko)):
            if x is None:
                continue
            x64 = x.double().cpu().numpy()
            ref = _ref64(x64, pos, turns, rot, inter, float(np.float32(mult)))
            err = np.abs(y.double().cpu().numpy() - ref)
            assert np.all(err <= _bound(x64, ref, rot, inter, mult, name)), float(err.max())


@pytest.mark.parametrize("scaling", [V.ROPE_PLAIN, V.ROPE_LINEAR, V.ROPE_NTK, V.ROPE_YARN])
@pytest.mark.parametrize("rot", [2, 64, 128])
def test_rope_turns_match_definition(scaling, rot):
    turns, mult = V.rope_turns(rot, 1e4, scaling, 8.0, 4096, 32.0, 1.0)
    f, m = _freqs64(rot, 1e4, scaling, 8.0, 4096, 32.0, 1.0)
    assert mult == np.float32(m)
    # a few roundings of 2^-53 in pow, log and the quotients
    assert np.allclose(turns.astype(np.float64) / 2.0 ** 64 * 2 * np.pi, f, rtol=1e-13, atol=2.0 ** -63)


def test_rope_strides_in_place_and_stream():
    """q and k as slices of a fused projection, rotated in place on a stream of their own; v is left alone."""
    torch = torch_cuda()
    rng = np.random.default_rng(3)
    t, hq, hk, d, rot = 19, 8, 2, 64, 32
    turns, mult = V.rope_turns(rot, 1e6)
    x = torch.from_numpy(rng.standard_normal((t, (hq + 2 * hk) * d))).float().cuda()
    before = x.clone()
    pos = rng.integers(0, 5000, size=t).astype(np.int32)
    dp, dt = torch.from_numpy(pos).cuda(), _turns_dev(torch, turns)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    row = x.shape[1]
    q, k = x.data_ptr(), x.data_ptr() + hq * d * 4
    V.rope(q, k, q, k, dp.data_ptr(), dt.data_ptr(), t, hq, hk, d, rot, q_stride=row, k_stride=row, q_out_stride=row,
           k_out_stride=row, stream=st.cuda_stream)
    st.synchronize()
    b64 = before.double().cpu().numpy().reshape(t, -1, d)
    ref = _ref64(b64[:, :hq + hk], pos, turns, rot, False, 1.0)
    got = x.double().cpu().numpy().reshape(t, -1, d)
    assert np.array_equal(got[:, hq + hk:], b64[:, hq + hk:])
    assert np.all(np.abs(got[:, :hq + hk] - ref) <= _bound(b64[:, :hq + hk], ref, rot, False, 1.0, "f32"))


def test_rope_unaligned_rows():
    """Odd token strides and a base off by one element: the one-element kernel."""
    torch = torch_cuda()
    rng = np.random.default_rng(4)
    t, hq, d, rot = 7, 3, 64, 64
    turns, _ = V.rope_turns(rot, 1e6)
    stride = hq * d + 3
    for name in ("f32", "f16"):
        dt = _torch_type(torch, name)
        buf = torch.from_numpy(rng.standard_normal(t * stride + 1)).to(dt).cuda()
        q = buf[1:].as_strided((t, hq, d), (stride, d, 1))
        pos = torch.arange(t, dtype=torch.int32, device="cuda") * 1000
        out = torch.empty((t, hq, d), dtype=dt, device="cuda")
        _call(torch, q, None, pos, _turns_dev(torch, turns), rot, name, False, 1.0, q_out=out, q_stride=stride)
        torch.cuda.synchronize()
        x64 = q.double().cpu().numpy()
        ref = _ref64(x64, pos.cpu().numpy(), turns, rot, False, 1.0)
        assert np.all(np.abs(out.double().cpu().numpy() - ref) <= _bound(x64, ref, rot, False, 1.0, name))


@pytest.mark.parametrize("inter", [False, True])
def test_rope_inverse_is_the_gradient(inter):
    """<rope(x), w> = <x, rope_inverse(w)> and central differences of <rope(x), w> in a few coordinates."""
    torch = torch_cuda()
    rng = np.random.default_rng(5 + inter)
    t, h, d, rot = 6, 3, 32, 24
    turns, mult = V.rope_turns(rot, 1e4, V.ROPE_YARN, 16.0, 64)
    pos = torch.from_numpy(rng.integers(0, 4096, size=t).astype(np.int32)).cuda()
    dt = _turns_dev(torch, turns)
    x = torch.from_numpy(rng.standard_normal((t, h, d)).astype(np.float32)).cuda()
    w = torch.from_numpy(rng.standard_normal((t, h, d)).astype(np.float32)).cuda()
    grad, _ = _call(torch, w, None, pos, dt, rot, "f32", inter, mult, inverse=True)

    def value(z):
        y, _ = _call(torch, z, None, pos, dt, rot, "f32", inter, mult)
        return float((y.double() * w.double()).sum())

    dot = float((x.double() * grad.double()).sum())
    # both sides carry errors of 5e-7 of each term
    terms = float((x.double().abs().sum() * 2 * mult * w.abs().max()))
    assert abs(value(x) - dot) <= 1e-6 * terms
    for at in [(0, 0, 0), (1, 1, 1), (3, 2, rot - 1), (5, 0, rot // 2), (2, 1, d - 1)]:
        step = torch.zeros_like(x)
        step[at] = 0.5
        diff = value(x + step) - value(x - step)
        assert abs(diff - float(grad[at])) <= 1e-6 * terms


def test_rope_offsets_past_32_bits():
    torch = torch_cuda()
    stride, d, rot = (1 << 30) + 8, 64, 64
    turns, _ = V.rope_turns(rot, 1e6)
    buf = torch.empty(2 * stride + 2 * stride // 2 + d, dtype=torch.float16, device="cuda")
    q = buf.as_strided((3, 1, d), (stride, d, 1))
    q.copy_(torch.randn((3, 1, d), device="cuda"))
    pos = torch.tensor([5, 70000, 123456], dtype=torch.int32, device="cuda")
    out = torch.empty((3, 1, d), dtype=torch.float16, device="cuda")
    _call(torch, q, None, pos, _turns_dev(torch, turns), rot, "f16", False, 1.0, q_out=out, q_stride=stride)
    torch.cuda.synchronize()
    x64 = q.double().cpu().numpy()
    ref = _ref64(x64, pos.cpu().numpy(), turns, rot, False, 1.0)
    assert np.all(np.abs(out.double().cpu().numpy() - ref) <= _bound(x64, ref, rot, False, 1.0, "f16"))
