"""Log probabilities, entropy and best alternatives against 64 bits: types, odd
vocabularies, ties, masks, infinities, NaN, empty rows, strides, temperatures."""
import math

import numpy as np
import pytest

import vspec_b200 as V
from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

DTYPES = {"f32": V.T_F32, "f16": V.T_F16, "bf16": V.T_BF16}

# A thread adds up to 600 values in fp32 (151936 over 512 threads, their rescales): the sum is off by at most
# 600 * 2^-24 + 2^-21 (the exponentials) = 3.7e-5 of itself, and so is ln of it; a log probability adds the
# rounding of its own terms.  U/(TS) carries the same error of its own size.
SUM = 3.7e-5


def _torch_type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _call(torch, x, name, tokens=None, top_k=0, allowed=None, inv_t=1.0, entropy=True, vocab=None, row_stride=0,
          rows=None, stream=0, workspace=None):
    rows, vocab = rows or x.shape[0], vocab or x.shape[1]
    n = tokens.shape[1] if tokens is not None else 0
    got = dict(lp=torch.full((rows, max(n, 1)), 9.0, device="cuda"), h=torch.full((rows,), 9.0, device="cuda"),
               top=torch.full((rows, max(top_k, 1)), 9.0, device="cuda"),
               ids=torch.full((rows, max(top_k, 1)), -9, dtype=torch.int32, device="cuda"))
    if stream:
        torch.cuda.synchronize()
    V.logprobs(x.data_ptr(), rows, vocab, DTYPES[name], tokens=tokens.data_ptr() if n else None, num_tokens=n,
               token_logprobs=got["lp"].data_ptr() if n else None, entropy=got["h"].data_ptr() if entropy else None,
               top_k=top_k, top_logprobs=got["top"].data_ptr() if top_k else None,
               top_ids=got["ids"].data_ptr() if top_k else None,
               allowed=allowed.data_ptr() if allowed is not None else None, inv_temperature=inv_t,
               row_stride=row_stride, stream=stream, workspace=workspace.data_ptr() if workspace is not None else None,
               workspace_bytes=workspace.numel() if workspace is not None else 0)
    torch.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in got.items()}


def _check(got, x, tokens, top_k, ok, inv_t, entropy=True):
    """x float64 [rows][vocab] on the host, ok bool or None."""
    for r in range(len(x)):
        v = x[r]
        allow = (np.ones(len(v), bool) if ok is None else ok[r]) & (v != -np.inf)
        live = v[allow]
        nan = bool(np.isnan(live).any() or (live == np.inf).any())
        if len(live) and not nan:
            m = live.max()
            e = np.exp((live - m) * inv_t)
            s = e.sum()
            lse, h = math.log(s), math.log(s) - float((e * (live - m)).sum()) * inv_t / s
            size = abs(h - math.log(s))
        order = np.flatnonzero(allow & ~np.isnan(v))
        order = order[np.lexsort((order, -v[order]))][:top_k] if top_k else []

        def want(i):
            if i < 0 or i >= len(v) or not allow[i]:
                return -np.inf
            return np.nan if nan else (v[i] - m) * inv_t - lse

        def same(a, b):
            if np.isnan(b):
                return np.isnan(a)
            if np.isinf(b):
                return a == b
            return abs(a - b) <= SUM + 4 * 2.0 ** -24 * abs(b)

        if tokens is not None:
            for i, a in zip(tokens[r], got["lp"][r]):
                assert same(a, want(int(i))), (r, i, a, want(int(i)))
        if entropy:
            if len(live) == 0:
                assert got["h"][r] == 0.0
            elif nan:
                assert np.isnan(got["h"][r])
            else:
                assert abs(got["h"][r] - h) <= SUM * (2 + 2 * size), (r, got["h"][r], h)
        if top_k:
            assert list(got["ids"][r][:len(order)]) == [int(i) for i in order]
            for i, a in zip(order, got["top"][r]):
                assert same(a, want(int(i)))
            assert (got["ids"][r][len(order):top_k] == -1).all()
            assert np.all(got["top"][r][len(order):top_k] == -np.inf)


def _bits(ok):
    rows, v = ok.shape
    pad = np.zeros((rows, -(-v // 32) * 32), dtype=bool)
    pad[:, :v] = ok
    return np.packbits(pad, axis=1, bitorder="little").view(np.int32)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top_k,n", [(1, 1, 1, 1), (3, 2, 5, 2), (2, 31, 32, 3), (5, 1000, 20, 8),
                                                (40, 4097, 7, 1), (4, 65537, 32, 4), (2, 151936, 20, 3),
                                                (700, 513, 3, 2), (3, 8191, 0, 5), (2, 20000, 1, 0)])
def test_matches_64_bit(name, rows, vocab, top_k, n):
    torch = torch_cuda()
    rng = np.random.default_rng(rows + vocab)
    x = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 3).to(_torch_type(torch, name)).cuda()
    tokens = rng.integers(0, vocab, size=(rows, n)).astype(np.int32) if n else None
    if n > 1:
        tokens[0, 0], tokens[-1, 1] = -1, vocab
    for inv_t in (1.0, 1.0 / 0.7):
        got = _call(torch, x, name, torch.from_numpy(tokens).cuda() if n else None, top_k, inv_t=inv_t)
        _check(got, x.double().cpu().numpy(), tokens, top_k, None, np.float64(np.float32(inv_t)))


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["up", "down", "flat", "steps"])
def test_ties_and_sorted_rows(name, order):
    """Ascending rows renew the whole list all the time; equal values go to the lowest ids."""
    torch = torch_cuda()
    vocab = 30011
    base = {"up": np.linspace(-5, 5, vocab), "down": np.linspace(5, -5, vocab), "flat": np.full(vocab, 1.25),
            "steps": np.repeat(np.arange(-(-vocab // 100)), 100)[:vocab] % 37 / 4.0}[order]
    x = torch.from_numpy(np.stack([base, -base]).astype(np.float32)).to(_torch_type(torch, name)).cuda()
    x[1, 17] = 0.0
    tokens = torch.tensor([[0, vocab - 1], [17, 5]], dtype=torch.int32, device="cuda")
    got = _call(torch, x, name, tokens, 32)
    _check(got, x.double().cpu().numpy(), tokens.cpu().numpy(), 32, None, 1.0)


def test_signed_zeros_tie():
    torch = torch_cuda()
    x = torch.full((1, 100), -1.0, device="cuda")
    x[0, 40], x[0, 60], x[0, 20] = -0.0, 0.0, 0.0
    got = _call(torch, x, "f32", None, 4)
    assert list(got["ids"][0]) == [20, 40, 60, 0]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [45, 1000, 9001])
def test_masks(name, vocab):
    """Allowed bits, with infinities and NaN where they are not set; rows with one allowed token and with none."""
    torch = torch_cuda()
    rng = np.random.default_rng(vocab)
    rows = 6
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    ok = rng.random((rows, vocab)) < 0.4
    ok[1] = False
    ok[1, vocab - 1] = True
    ok[2] = False
    ok[3] = True
    x[~ok] = rng.choice([np.nan, np.inf, -np.inf, 65504.0, -65504.0], size=int((~ok).sum()))
    x[4, ok[4]] = -np.inf                                   # allowed, and all of them -inf
    xt = torch.from_numpy(x).to(_torch_type(torch, name)).cuda()
    tokens = rng.integers(0, vocab, size=(rows, 6)).astype(np.int32)
    tokens[1, 0] = vocab - 1
    got = _call(torch, xt, name, torch.from_numpy(tokens).cuda(), 32, allowed=torch.from_numpy(_bits(ok)).cuda())
    _check(got, xt.double().cpu().numpy(), tokens, 32, ok, 1.0)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_infinities_nan_and_lowest_values(name):
    torch = torch_cuda()
    vocab = 5000
    rng = np.random.default_rng(9)
    x = rng.standard_normal((7, vocab)).astype(np.float32)
    xt = torch.from_numpy(x).to(_torch_type(torch, name)).cuda()
    low = torch.finfo(xt.dtype).min
    xt[0, 33] = float("nan")
    xt[1, 44] = float("inf")
    xt[2] = float("-inf")
    xt[3, 1:] = low
    xt[4] = low                                            # a row of the type's lowest value is uniform
    xt[5, ::2] = float("-inf")
    xt[6, 4999] = torch.finfo(xt.dtype).max
    tokens = torch.tensor([[33, 2]] * 7, dtype=torch.int32, device="cuda")
    tokens[1, 0], tokens[6, 0], tokens[3, 0] = 44, 4999, 0
    got = _call(torch, xt, name, tokens, 10)
    _check(got, xt.double().cpu().numpy(), tokens.cpu().numpy(), 10, None, 1.0)


def test_strided_rows_stream_and_offsets_past_32_bits():
    torch = torch_cuda()
    rng = np.random.default_rng(10)
    vocab = 777
    for stride in (vocab + 5, 1 << 30):
        buf = torch.empty(2 * stride + vocab, dtype=torch.float16, device="cuda") if stride > 10000 else \
            torch.zeros(2 * stride + vocab, dtype=torch.float16, device="cuda")
        x = buf.as_strided((3, vocab), (stride, 1))
        x.copy_(torch.from_numpy(rng.standard_normal((3, vocab)).astype(np.float32)))
        tokens = torch.tensor([[1], [776], [300]], dtype=torch.int32, device="cuda")
        st = torch.cuda.Stream()
        got = _call(torch, x, "f16", tokens, 5, row_stride=stride, stream=st.cuda_stream)
        _check(got, x.double().cpu().numpy(), tokens.cpu().numpy(), 5, None, 1.0)


def test_split_rows_share_a_workspace():
    """Few long rows are split over CTAs; calls of several shapes share one zero-filled workspace and stay exact
    call after call."""
    torch = torch_cuda()
    rng = np.random.default_rng(12)
    shapes = [(2, 151936, 20), (9, 40000, 5), (1, 65537, 32)]
    need = max(V.lib.vspec_b200_logprobs_workspace_bytes(*s) for s in shapes)
    ws = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        for rows, vocab, k in shapes:
            x = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32)).cuda()
            first = _call(torch, x, "f32", None, k, workspace=ws)
            _check(first, x.double().cpu().numpy(), None, k, None, 1.0)
            again = _call(torch, x, "f32", None, k, workspace=ws)
            assert all(np.array_equal(first[n], again[n]) for n in first)
    with pytest.raises(V.VspecB200Error, match="workspace"):
        _call(torch, x, "f32", None, 32, workspace=ws[:1024])


def test_workspace_of_any_contents():
    """What a caller's workspace held before does not matter."""
    torch = torch_cuda()
    rows, vocab, k = 3, 50001, 7
    x = torch.randn((rows, vocab), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    ws = torch.empty(V.lib.vspec_b200_logprobs_workspace_bytes(rows, vocab, k), dtype=torch.uint8, device="cuda")
    assert ws.numel() > 0
    expect = _call(torch, x, "f32", None, k)
    for fill in (0xFF, 0x01, 0x00):
        ws.fill_(fill)
        got = _call(torch, x, "f32", None, k, workspace=ws)
        torch.cuda.synchronize()
        assert all(np.array_equal(got[n], expect[n]) for n in got)
