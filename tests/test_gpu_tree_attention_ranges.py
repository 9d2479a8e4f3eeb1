"""Tree attention at the ends of its inputs' ranges, in the kernel for few rows
and in the one for many, and what else the two have to share: streams, host
threads, graphs, offsets, heads."""
import threading

import numpy as np
import pytest

import vspec_b200 as V
from gpu_util import torch_cuda
from test_gpu_tree_attention import BOUND, MANY, Case, _torch_type, _widen_table

pytestmark = pytest.mark.gpu

KERNELS = ["few rows", "many rows"]


def _case(kernel, ctx, trees, kv, name, seed, hq=8, hkv=2, d=128, pt=16, **kw):
    """A case whose plan takes the kernel: 17 to 64 rows a pair go to the one for many rows with a table that
    could hold a long context, else to the other."""
    torch = torch_cuda()
    case = Case(torch, np.random.default_rng(seed), ctx, trees, hq, hkv, d, pt, kv, name, **kw)
    rows = case.max_q * hq // hkv
    assert 16 < rows <= 64 and -(-rows // 16) * case.batch * hkv * case.max_ctx < 1 << 18
    if kernel == "many rows":
        _widen_table(case, MANY)
        case.max_ctx = MANY
    return case


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_results_are_rounded_once(kernel, kv, name):
    """16-bit queries and results: the error is that of rounding the exact result, within 1.1 for the chance of
    which values are near a tie, and what fp32 holds: weights within 2e-5 (scores within 1e-5), so a result
    within that of sum p |v|."""
    case = _case(kernel, [30, 9, 61, 250], [6, 8, 5, 7], kv, name, 101)
    out = case.run().double()
    case.torch.cuda.synchronize()
    ref, _ = case.ref()
    signed = case.codes[1]
    if kv == "f16":
        case.codes[1] = signed.abs()
    elif kv == "fp8":
        case.codes[1] = signed & 0x7F
    else:
        case.codes[1] = signed.view(case.torch.int8).abs().view(case.torch.uint8)
    size, _ = case.ref()
    once = (ref.to(_torch_type(case.torch, name)).double() - ref).norm().item()
    err = (out - ref).norm().item()
    print(f"{kernel} {kv} {name}: {err / ref.norm().item():.3e}, rounded once {once / ref.norm().item():.3e}")
    assert err <= 1.1 * once + 2e-5 * size.norm().item()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("ctx,n,hq,hkv,d", [([0], 900, 4, 4, 64), ([50, 200], 400, 4, 2, 128), ([13], 640, 2, 1, 128)])
def test_long_chunks_over_fp16_pages(name, ctx, n, hq, hkv, d):
    """A prompt's chunk over many steps of 128 tokens, each of them with drafted tokens."""
    case = Case(torch_cuda(), np.random.default_rng(n), ctx, [n] * len(ctx), hq, hkv, d, 16, "f16", name)
    case.causal = True
    case.check(case.run(use_cu=False))
    assert V.tree_attention_timeout_flag() == 0


@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
def test_waits_that_give_up_are_told_and_leave_nothing_behind(kv):
    """With a limit of no time a call's waits may give up at once: then the flag says so, else the result is whole.
    The calls after it are right."""
    torch = torch_cuda()
    case = Case(torch, np.random.default_rng(103), [6000, 3000], [40, 33], 8, 2, 128, 16, kv, "f32")
    expect = case.run().clone()
    torch.cuda.synchronize()
    assert V.tree_attention_timeout_flag() == 0
    gave_up = 0
    try:
        V.check(V.lib.vspec_b200_debug_tree_wait_cycles(0))
        for _ in range(10):
            out = case.run()
            torch.cuda.synchronize()
            flag = V.tree_attention_timeout_flag()
            assert flag or torch.equal(out, expect)
            gave_up += flag
    finally:
        V.check(V.lib.vspec_b200_debug_tree_wait_cycles(-1))
    print(f"{kv}: {gave_up} of 10 calls gave up")
    assert torch.equal(case.run(), expect) and V.tree_attention_timeout_flag() == 0


def _slots(case, b, t):
    """Pool rows of sequence b's tokens t."""
    t = np.asarray(t)
    return case.torch.from_numpy(case.table[b, t // case.pt].astype(np.int64) * case.pt + t % case.pt).cuda()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("zeros", [(0, 128), (0, 300), (128, 1100), (0, 1999)])
def test_v_rows_of_zeros_count_in_the_sum(kernel, kv, zeros):
    """V rows of zeros have scale 0; their tokens weigh as much as others."""
    case = _case(kernel, [2000, 1990, 1500, 700], [8, 5, 7, 6], kv, "f32", 104, hq=32, hkv=8)
    for b, c in enumerate(case.ctx):
        at = _slots(case, b, np.arange(zeros[0], min(zeros[1], c)))
        case.codes[1][at] = 0
        case.scales[1][at] = 0.0
    case.check(case.run())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "f16"])
def test_committed_values_that_are_not_finite_reach_every_row(kernel, kv, name):
    """NaN and infinities in V (codes or scales) of a committed token make results non-finite where the definition
    does, also when the token shares its step with drafted ones."""
    torch = torch_cuda()
    for t, what in ((70, "nan"), (150, "inf"), (290, "inf"), (20, "nan")):
        case = _case(kernel, [300, 160], [6, 7], kv, name, 105)
        at = _slots(case, 0 if t > 160 else 1, [t])
        value = float(what)
        if kv == "f16":
            case.codes[1][at, 0, 5::16] = value
        elif kv == "fp8" and what == "nan":
            case.codes[1][at, 0, 5::16] = 0x7F
        else:
            case.scales[1][at, 0] = value
        got = case.run().double()
        torch.cuda.synchronize()
        ref, _ = case.ref()
        fine = torch.isfinite(ref)
        assert not fine.all() and fine.any()
        if kv != "f16" and what == "inf":      # a code of 0 times the scale is NaN, any other an infinity
            assert not torch.isfinite(got[~fine]).any()
        else:
            assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(torch.isinf(got), torch.isinf(ref))
        top = float(torch.nan_to_num(torch.cat([case.rows64(1, b, c + n).flatten() for b, (c, n) in
                                                enumerate(zip(case.ctx, case.trees))]), 0, 0, 0).abs().max())
        assert (got - ref)[fine].abs().max().item() <= BOUND[name] * top


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "f16"])
@pytest.mark.parametrize("power", [20, 40, 60, 100])
def test_large_v_scales_that_are_not_seen_do_not_reach_a_row(kernel, kv, name, power):
    """V scales of drafted tokens 2^power times the others': rows that do not see them are as without them, bit
    for bit, and rows that do are right, in a tree behind a context and in a chunk at the start of one."""
    torch = torch_cuda()
    for ctx, causal in (([75, 130], False), ([0, 3], True)):
        case = _case(kernel, ctx, [12, 9], kv, name, 106)
        case.causal = causal
        bad = {0: [7], 1: [5, 6]}
        if not causal:
            for b, row in ((0, 0), (1, 12)):
                for j in bad[b]:
                    case.bits[row:row + case.trees[b], 0] &= ~np.uint32(1 << j)
        clean = case.run().clone()
        case.check(clean)
        if not causal:
            case.bits[3, 0] |= np.uint32(1 << 7)
            case.bits[12 + 8, 0] |= np.uint32(1 << 5)
        for b in bad:
            case.scales[1][_slots(case, b, [ctx[b] + j for j in bad[b]])] *= 2.0 ** power
        got = case.run()
        sees = list(range(7, 12)) + list(range(12 + 5, 12 + 9)) if causal else [3, 12 + 8]
        rest = [i for i in range(21) if i not in sees]
        torch.cuda.synchronize()
        assert torch.equal(got[rest], clean[rest])
        if name == "f32":                    # fp16 results end at 65504
            case.check(got)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kv", ["f16", "int8"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("power", [110, 120, -110])
def test_queries_at_the_ends_of_their_range(kernel, kv, name, power):
    """Queries of 2^power: with a scale to match the scores are ordinary ones."""
    case = _case(kernel, [90, 40], [6, 8], kv, name, 107)
    case.q = (case.q.double() * 2.0 ** power).to(case.q.dtype)
    case.scale *= 2.0 ** -power
    case.check(case.run())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kv", ["fp8", "int8"])
@pytest.mark.parametrize("order", ["up", "down"])
def test_uneven_v_scales(kernel, kv, order):
    """V scales over thirty orders of magnitude along the context."""
    torch = torch_cuda()
    case = _case(kernel, [640, 900], [8, 5], kv, "f32", 112)
    for b, (c, n) in enumerate(zip(case.ctx, case.trees)):
        scales = torch.logspace(-20, 10, c + n, device="cuda").unsqueeze(-1)
        case.scales[1][_slots(case, b, np.arange(c + n))] = scales if order == "up" else scales.flip(0)
    case.check(case.run())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kv", ["f16", "fp8"])
def test_graph_replays_follow_lengths(kernel, kv):
    torch = torch_cuda()
    case = _case(kernel, [500, 40], [6, 8], kv, "f16", 113)
    need = V.lib.vspec_b200_tree_attention_workspace_bytes(2, case.total, 8, 8, 2, 128, case.max_ctx)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    out = case.run(workspace=ws)
    torch.cuda.synchronize()
    table, ctx, cu, mask = case._keep
    scales = [s.data_ptr() if s is not None else None for s in case.scales]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        V.tree_attention(case.q.data_ptr(), case.codes[0].data_ptr(), case.codes[1].data_ptr(), *scales,
                         table.data_ptr(), ctx.data_ptr(), cu.data_ptr(), mask.data_ptr(), out.data_ptr(), 2, case.total,
                         8, 8, 2, 128, 16, case.table.shape[1], case.pages, case.max_ctx, case.scale, q_dtype=V.T_F16,
                         kv_dtype=V.KV_F16 if kv == "f16" else V.KV_FP8, mask_words=case.words,
                         workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                         stream=torch.cuda.current_stream().cuda_stream)
    for ctx_now, trees_now in (([500, 40], [6, 8]), ([7, 41], [8, 4]), ([300, 0], [6, 8]), ([127, 128], [1, 2])):
        case.ctx, case.trees = ctx_now, trees_now
        ctx.copy_(torch.tensor(ctx_now, dtype=torch.int32))
        cu.copy_(torch.tensor([0] + list(np.cumsum(trees_now)), dtype=torch.int32))
        g.replay()
        out[sum(trees_now):] = 0
        total, case.total = case.total, sum(trees_now)
        q, case.q = case.q, case.q[:case.total]
        case.check(out[:case.total])
        case.total, case.q = total, q


@pytest.mark.parametrize("kernel", KERNELS)
def test_streams_and_host_threads(kernel):
    """Two host threads, each on a stream of its own with the library's scratch, time and again."""
    torch = torch_cuda()
    cases = [_case(kernel, [900, 350], [8, 5], "f16", "f32", 114), _case(kernel, [300, 800], [6, 7], "fp8", "f32", 115)]
    expect = [c.run().clone() for c in cases]
    torch.cuda.synchronize()
    got, wrong = [None, None], []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    got[i] = cases[i].run(stream=st.cuda_stream)
                    st.synchronize()
                    if not torch.equal(got[i], expect[i]):
                        wrong.append(i)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for c, out in zip(cases, expect):
        c.check(out)


@pytest.mark.parametrize("kv", ["f16", "int8"])
def test_pool_offsets_past_32_bits_many_rows(kv):
    """Pages beyond 2^31 elements of the pool."""
    torch = torch_cuda()
    case = _case("many rows", [100], [24], kv, "f32", 116, hq=8, hkv=8)
    far = (1 << 31) // (16 * 8 * 128) + 5
    rows = far * 16
    pool = torch.empty((rows + case.codes[0].shape[0], 8, 128), dtype=case.codes[0].dtype, device="cuda")
    pool[rows:] = case.codes[0]
    case.codes = [pool, pool]
    if kv != "f16":
        wide = torch.empty((rows + case.scales[0].shape[0], 8), device="cuda")
        wide[rows:] = case.scales[0]
        case.scales = [wide, wide]
    case.table = np.where(case.table >= 0, case.table + far, case.table).astype(np.int32)
    case.pages += far
    case.check(case.run())


@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("trees", [[4, 2], [9, 3], [20, 7]])
def test_heads_of_256(kv, name, trees):
    """One, two and four row warps."""
    case = Case(torch_cuda(), np.random.default_rng(117), [333, 64], trees, 8, 4, 256, 16, kv, name)
    case.check(case.run())


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
def test_repeated_calls_are_identical(kernel, kv):
    torch = torch_cuda()
    case = _case(kernel, [1500, 1200], [8, 7], kv, "bf16", 118)
    first = case.run().clone()
    for _ in range(10):
        assert torch.equal(case.run(), first)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kv", ["f16", "int8"])
@pytest.mark.parametrize("length", [1 << 20, (1 << 31) - 1])
def test_lengths_past_the_page_table_are_told(kernel, kv, length):
    """The flag is raised, and the other sequences are right."""
    torch = torch_cuda()
    case = _case(kernel, [500, 40], [6, 8], kv, "f32", 108)
    ref, big = case.ref()
    V.page_fault_flag()
    case.ctx = [length, 40]
    got = case.run()
    torch.cuda.synchronize()
    assert V.page_fault_flag() == 1 and V.tree_attention_timeout_flag() == 0
    assert ((got.double() - ref).abs() / big)[6:].max().item() <= BOUND["f32"]


@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d", [48, 64, 80, 128])
def test_more_rows_than_a_tile(kv, name, d):
    """129 to 280 rows a pair: one or two row tiles a CTA."""
    case = Case(torch_cuda(), np.random.default_rng(119), [700, 0, 130], [33, 43, 70], 8, 2, d, 16, kv, name)
    case.check(case.run())
