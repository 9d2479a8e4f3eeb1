"""Attention of drafted-token trees over paged caches against a plain 64-bit
implementation: page types, query types, head layouts, tree and context sizes
from nothing to many pages, masks that hide whole rows, values that a row must
not see, strides, streams, graphs, and agreement with the decode attention."""
import math

import numpy as np
import pytest

import vspec_b200 as V
from gpu_util import torch_cuda

pytestmark = pytest.mark.gpu

DTYPES = {"f32": V.T_F32, "f16": V.T_F16, "bf16": V.T_BF16}
KINDS = {"f16": V.KV_F16, "fp8": V.KV_FP8, "int8": V.KV_INT8}

# Normwise bounds, over the largest |V| a row sees.  fp32: a score is off by at most |q||k| scale * 2^-20 (split
# products 2^-22, 128 fp32 additions), about 1e-5 for these inputs, so a weight by twice that.  16-bit: weights
# rounded to fp16 (2^-11 at most) and the result's own half ulp, 2^-11 or 2^-8.
BOUND = {"f32": 4e-5, "f16": 2 * 2.0 ** -11 + 4e-5, "bf16": 2.0 ** -11 + 2.0 ** -8 + 4e-5}


def _torch_type(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _random_tree_bits(rng, n, words):
    bits = np.zeros((n, words), dtype=np.uint32)
    for j in range(n):
        parent = int(rng.integers(-1, j)) if j else -1
        if parent >= 0:
            bits[j] = bits[parent]
        bits[j, j // 32] |= np.uint32(1 << (j % 32))
    return bits


class Case:
    def __init__(self, torch, rng, ctx, trees, hq, hkv, d, pt, kv, name, max_q=None, spare=2, scale=None, magnitude=1.0):
        self.torch, self.ctx, self.trees = torch, ctx, trees
        self.hq, self.hkv, self.d, self.pt, self.kv, self.name = hq, hkv, d, pt, kv, name
        self.batch, self.total = len(ctx), sum(trees)
        self.max_q = max_q or max(max(trees), 1)
        self.words = -(-self.max_q // 32)
        lens = [c + n for c, n in zip(ctx, trees)]
        need = [-(-n // pt) for n in lens]
        self.pages = sum(need) + spare
        perm = rng.permutation(self.pages).astype(np.int32)
        self.table = np.zeros((self.batch, max(max(need), 1)), dtype=np.int32)
        o = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[o:o + n]
            o += n
        g = torch.Generator(device="cuda")
        g.manual_seed(int(rng.integers(1 << 30)))
        rows = self.pages * pt
        self.codes, self.scales = [], []
        kvf = [torch.randn((rows, hkv, d), device="cuda", generator=g) * magnitude for _ in range(2)]
        if kv == "f16":
            self.codes = [x.half() for x in kvf]
            self.scales = [None, None]
        else:
            kvf[1] *= torch.exp(torch.randn((rows, hkv, 1), device="cuda", generator=g))   # uneven V scales
            c = [torch.empty((rows, hkv, d), dtype=torch.uint8, device="cuda") for _ in range(2)]
            s = [torch.empty((rows, hkv), device="cuda") for _ in range(2)]
            V.kv_quant_append(kvf[0].data_ptr(), kvf[1].data_ptr(), None, rows, hkv, d, rows, KINDS[kv],
                              c[0].data_ptr(), c[1].data_ptr(), s[0].data_ptr(), s[1].data_ptr())
            self.codes, self.scales = c, s
        self.q = torch.randn((self.total, hq, d), device="cuda", generator=g).to(_torch_type(torch, name))
        self.bits = np.zeros((self.total, self.words), dtype=np.uint32)
        row = 0
        for n in trees:
            self.bits[row:row + n] = _random_tree_bits(rng, n, self.words)
            row += n
        self.causal = False
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale
        self.max_ctx = max(lens)

    def run(self, stream=0, out=None, use_cu=True, workspace=None, q=None, q_stride=0, max_ctx=None, batch=None):
        torch = self.torch
        dev = "cuda"
        self._keep = [torch.from_numpy(self.table).to(dev), torch.tensor(self.ctx, dtype=torch.int32, device=dev),
                      torch.tensor([0] + list(np.cumsum(self.trees)), dtype=torch.int32, device=dev),
                      torch.from_numpy(self.bits.view(np.int32).copy()).to(dev)]
        table, ctx, cu, mask = self._keep
        if out is None:
            out = torch.full((self.total, self.hq, self.d), 7.0, dtype=self.q.dtype, device=dev)
        if stream:
            torch.cuda.synchronize()
        V.tree_attention((self.q if q is None else q).data_ptr(), self.codes[0].data_ptr(), self.codes[1].data_ptr(),
                         self.scales[0].data_ptr() if self.scales[0] is not None else None,
                         self.scales[1].data_ptr() if self.scales[1] is not None else None, table.data_ptr(),
                         ctx.data_ptr(), cu.data_ptr() if use_cu else None,
                         None if self.causal else mask.data_ptr(), out.data_ptr(), self.batch, self.total, self.max_q,
                         self.hq, self.hkv, self.d, self.pt, self.table.shape[1], self.pages,
                         self.max_ctx if max_ctx is None else max_ctx, self.scale, q_dtype=DTYPES[self.name],
                         kv_dtype=KINDS[self.kv], mask_words=self.words, q_stride=q_stride,
                         workspace=workspace.data_ptr() if workspace is not None else None,
                         workspace_bytes=workspace.numel() if workspace is not None else 0, stream=stream)
        return out

    def rows64(self, which, b, n):
        torch = self.torch
        t = np.arange(n)
        slot = torch.from_numpy(self.table[b, t // self.pt].astype(np.int64) * self.pt + t % self.pt).cuda()
        c = self.codes[which][slot]
        if self.kv == "f16":
            return c.double()
        c = c.view(torch.int8) if self.kv == "int8" else c.view(torch.float8_e4m3fn)
        return c.double() * self.scales[which][slot].double().unsqueeze(-1)

    def ref(self):
        """Softmax over what a row sees alone: what it does not see never enters the arithmetic."""
        torch = self.torch
        out = torch.zeros((self.total, self.hq, self.d), dtype=torch.float64, device="cuda")
        big = torch.zeros((self.total, self.hq, 1), dtype=torch.float64, device="cuda")
        row, group = 0, self.hq // self.hkv
        for b, (c, n) in enumerate(zip(self.ctx, self.trees)):
            if n == 0:
                continue
            k, v = self.rows64(0, b, c + n), self.rows64(1, b, c + n)
            for i in range(n):
                see = [j <= i if self.causal else bool(self.bits[row + i, j // 32] >> (j % 32) & 1) for j in range(n)]
                at = torch.tensor(list(range(c)) + [c + j for j in range(n) if see[j]], dtype=torch.long, device="cuda")
                if len(at):
                    qq = self.q[row + i].double().view(self.hkv, group, self.d)
                    s = torch.einsum("hgd,thd->hgt", qq, k[at]) * self.scale
                    out[row + i] = torch.einsum("hgt,thd->hgd", torch.softmax(s, -1), v[at]).reshape(self.hq, self.d)
                    big[row + i] = v[at].abs().amax((0, 2)).repeat_interleave(group).unsqueeze(-1)
            row += n
        return out, big

    def check(self, out, times=1.0):
        self.torch.cuda.synchronize()
        assert V.page_fault_flag() == 0
        ref, big = self.ref()
        err = ((out.double() - ref).abs() / big.clamp_min(1e-30)).max().item() if self.total else 0.0
        assert self.torch.isfinite(out.double()).all()
        print(f"ctx={self.ctx} trees={self.trees} {self.hq}/{self.hkv}x{self.d} {self.kv} {self.name}: {err:.2e}")
        assert err <= BOUND[self.name] * times
        empty = (big == 0).expand_as(ref)
        assert (out[empty] == 0).all()


@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ctx,trees,hq,hkv,d,pt", [
    ([5], [1], 1, 1, 128, 16),                              # one token, one head
    ([0, 1, 63, 64, 65], [1, 3, 2, 5, 1], 4, 2, 128, 16),   # around a step of 64 tokens
    ([37, 300, 0], [8, 0, 4], 32, 8, 128, 16),              # an empty tree, an empty context
    ([129, 700], [13, 7], 16, 2, 64, 5),                    # pages that end inside a step
    ([1000], [33], 8, 8, 128, 16),                          # two mask words
    ([250, 90], [40, 64], 8, 4, 96, 24),                    # a head size between the kernels'
    ([130], [6], 6, 2, 256, 16),                            # a group of three
    ([17], [70], 5, 1, 16, 1),                              # three mask words, one-token pages
    ([3000], [2], 7, 7, 128, 64),                           # several context pieces
    ([600, 20, 4100], [20, 64, 31], 64, 8, 128, 16),        # many rows a pair
])
def test_matches_64_bit(kv, name, ctx, trees, hq, hkv, d, pt):
    torch = torch_cuda()
    case = Case(torch, np.random.default_rng(sum(ctx) + hq + d), ctx, trees, hq, hkv, d, pt, kv, name)
    case.check(case.run())


@pytest.mark.parametrize("kv", ["f16", "int8"])
@pytest.mark.parametrize("d", [8, 40, 72, 136, 200, 248])
def test_odd_head_sizes(kv, d):
    torch = torch_cuda()
    if kv == "int8" and d % 16:
        d = d // 16 * 16 + 16
    case = Case(torch, np.random.default_rng(d), [77, 200], [5, 9], 4, 2, d, 16, kv, "f32")
    case.check(case.run())


@pytest.mark.parametrize("kv", ["f16", "fp8"])
@pytest.mark.parametrize("name", ["f32", "f16"])
def test_chain_without_mask(kv, name):
    """No mask and no d_cu_q: drafted tokens see each other up to themselves (a chunk of a prompt)."""
    torch = torch_cuda()
    for ctx, n in (([0, 0], 48), ([100, 640], 7), ([31], 256)):
        case = Case(torch, np.random.default_rng(n), ctx, [n] * len(ctx), 8, 2, 128, 16, kv, name)
        case.causal = True
        case.check(case.run(use_cu=False))


def test_single_tokens_agree_with_decode_attention():
    """One drafted token a sequence is the decode attention over ctx + 1 tokens."""
    torch = torch_cuda()
    ctx = [36, 299, 1500]
    case = Case(torch, np.random.default_rng(11), ctx, [1, 1, 1], 32, 8, 128, 16, "f16", "f32")
    out = case.run()
    ref = torch.empty_like(out)
    table = torch.from_numpy(case.table).cuda()
    lens = torch.tensor([c + 1 for c in ctx], dtype=torch.int32, device="cuda")
    V.paged_attention(case.q.data_ptr(), case.codes[0].data_ptr(), case.codes[1].data_ptr(), table.data_ptr(),
                      lens.data_ptr(), ref.data_ptr(), 3, 32, 8, 128, 16, case.table.shape[1], case.pages, max(ctx) + 1,
                      case.scale)
    torch.cuda.synchronize()
    assert (out - ref).abs().max().item() <= 2 * BOUND["f32"] * float(case.codes[1].abs().max())


@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("ctx", [0, 90])
def test_rows_that_see_nothing_or_not_themselves(kv, ctx):
    torch = torch_cuda()
    case = Case(torch, np.random.default_rng(21 + ctx), [ctx, ctx], [9, 40], 8, 2, 128, 16, kv, "f32")
    case.bits[0] = 0
    case.bits[8] = 0
    case.bits[9:30] = 0
    case.bits[31, 0] = 1 << 2            # another token only
    case.bits[33] = 0xFFFFFFFF           # bits past the tree's 40 tokens are ignored
    case.check(case.run())


@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("hq", [4, 32])
def test_values_that_are_not_seen_do_not_reach_a_row(kv, name, hq):
    """NaN and infinities in K, V and scales of drafted tokens: rows that do not see them are as without
    them, rows that do are not finite.  Slots past the last token hold NaN throughout."""
    torch = torch_cuda()
    ctx, n = 75, 12
    case = Case(torch, np.random.default_rng(31), [ctx], [n], hq, 2, 128, 16, kv, name)
    bad = [3, 7]
    for i in range(n):
        for j in bad:
            case.bits[i, 0] &= ~np.uint32(1 << j)
    clean = case.run().clone()
    case.check(clean)
    t = np.arange(ctx + n, case.table.shape[1] * 16)
    slot = torch.from_numpy(case.table[0, t // 16].astype(np.int64) * 16 + t % 16).cuda()
    at = [int(case.table[0, (ctx + j) // 16]) * 16 + (ctx + j) % 16 for j in bad]
    for c, s in zip(case.codes, case.scales):
        if kv == "f16":
            c[slot] = float("nan")
            c[at[0]] = float("nan")
            c[at[1], :, ::3] = float("inf")
        else:
            s[slot] = float("nan")
            s[at[0]] = float("nan")
            s[at[1]] = float("inf")
            if kv == "fp8":
                c[slot] = 0x7F
                c[at[1]] = 0x7F
    got = case.run()
    torch.cuda.synchronize()
    assert torch.equal(got, clean)
    case.bits[5, 0] |= np.uint32(1 << bad[0])
    case.bits[6, 0] |= np.uint32(1 << bad[1])
    got = case.run()
    torch.cuda.synchronize()
    finite = torch.isfinite(got.double()).all(-1)
    assert not finite[5].any() and not torch.isfinite(got[6].double()).all(-1).any()
    rest = [i for i in range(n) if i not in (5, 6)]
    assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("kv", ["f16", "int8"])
def test_large_and_small_scores(kv):
    """Scores far from 0, a scale of 0 and a negative one."""
    torch = torch_cuda()
    for scale, magnitude in ((3.0, 1.0), (0.0, 1.0), (-0.2, 1.0), (0.01, 1e-3), (1e-5, 100.0)):
        case = Case(torch, np.random.default_rng(5), [200], [10], 4, 1, 64, 16, kv, "f32", scale=scale,
                    magnitude=magnitude)
        # |q||k| scale reaches 64 * 3: the score bound grows with it
        case.check(case.run(), times=max(1.0, 12 * abs(scale) * magnitude))


def test_uneven_v_scales_keep_precision():
    """V scales over thirty orders of magnitude, ascending and descending along the context."""
    torch = torch_cuda()
    for order in (1, -1):
        case = Case(torch, np.random.default_rng(6), [640], [4], 4, 1, 128, 16, "int8", "f32")
        t = np.arange(644)
        slot = torch.from_numpy(case.table[0, t // 16].astype(np.int64) * 16 + t % 16).cuda()
        case.scales[1][slot] = torch.logspace(-20, 10, 644, device="cuda")[::order].unsqueeze(-1) if order == 1 else \
            torch.logspace(-20, 10, 644, device="cuda").flip(0).unsqueeze(-1)
        case.check(case.run())


def test_strided_queries_stream_and_workspace():
    torch = torch_cuda()
    rng = np.random.default_rng(41)
    case = Case(torch, rng, [900, 350], [11, 5], 8, 2, 128, 16, "f16", "f32")
    row = (8 + 4) * 128
    wide = torch.randn((case.total, row), device="cuda")
    wide[:, :8 * 128] = case.q.reshape(case.total, -1)
    st = torch.cuda.Stream()
    need = V.lib.vspec_b200_tree_attention_workspace_bytes(2, case.total, 11, 8, 2, 128, case.max_ctx)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = case.run(stream=st.cuda_stream, q=wide, q_stride=row, workspace=ws)
    st.synchronize()
    case.check(out)
    with pytest.raises(V.VspecB200Error, match="workspace"):
        case.run(workspace=ws[:need - 16])
    case.check(case.run(max_ctx=0))                 # the table's capacity bounds the plan


def test_graph_replay_with_new_lengths():
    """A captured call reads lengths, trees and masks from the device: replays follow them."""
    torch = torch_cuda()
    case = Case(torch, np.random.default_rng(51), [500, 40], [6, 3], 8, 2, 128, 16, "int8", "f16")
    need = V.lib.vspec_b200_tree_attention_workspace_bytes(2, case.total, 6, 8, 2, 128, case.max_ctx)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    out = case.run(workspace=ws)
    torch.cuda.synchronize()
    table, ctx, cu, mask = case._keep
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        V.tree_attention(case.q.data_ptr(), case.codes[0].data_ptr(), case.codes[1].data_ptr(),
                         case.scales[0].data_ptr(), case.scales[1].data_ptr(), table.data_ptr(), ctx.data_ptr(),
                         cu.data_ptr(), mask.data_ptr(), out.data_ptr(), 2, case.total, 6, 8, 2, 128, 16,
                         case.table.shape[1], case.pages, case.max_ctx, case.scale, q_dtype=V.T_F16, kv_dtype=V.KV_INT8,
                         mask_words=case.words, workspace=ws.data_ptr(), workspace_bytes=ws.numel(),
                         stream=torch.cuda.current_stream().cuda_stream)
    for ctx_now, trees_now in (([500, 40], [6, 3]), ([7, 41], [5, 4]), ([300, 0], [3, 6])):
        case.ctx, case.trees = ctx_now, trees_now
        ctx.copy_(torch.tensor(ctx_now, dtype=torch.int32))
        cu.copy_(torch.tensor([0] + list(np.cumsum(trees_now)), dtype=torch.int32))
        g.replay()
        case.check(out)


def test_repeated_calls_are_identical():
    torch = torch_cuda()
    case = Case(torch, np.random.default_rng(61), [3000, 1200], [16, 16], 32, 8, 128, 16, "fp8", "f32")
    first = case.run().clone()
    for _ in range(3):
        assert torch.equal(case.run(), first)


def test_pool_offsets_past_32_bits():
    """Pages beyond 2^31 elements of the pool."""
    torch = torch_cuda()
    case = Case(torch, np.random.default_rng(71), [100], [4], 8, 8, 128, 16, "f16", "f32")
    far = (1 << 31) // (16 * 8 * 128) + 5
    pool = torch.empty(((far + case.pages) * 16, 8, 128), dtype=torch.float16, device="cuda")
    pool[far * 16:] = case.codes[0]
    case.codes = [pool, pool]
    case.table = case.table + far
    case.pages += far
    case.check(case.run())


def test_bad_page_raises_the_flag():
    torch = torch_cuda()
    case = Case(torch, np.random.default_rng(81), [40], [4], 4, 1, 128, 16, "f16", "f32")
    case.table[0, 1] = case.pages
    V.page_fault_flag()
    case.run()
    torch.cuda.synchronize()
    assert V.page_fault_flag() == 1


# The plan takes lengths from max_ctx, so a small case reaches the kernel for many rows through a large one,
# which needs a page table that could hold it; what the table has past a sequence's pages is not looked at.
MANY = 1 << 18


def _widen_table(case, tokens):
    extra = np.full((case.batch, max(-(-tokens // case.pt) - case.table.shape[1], 0)), -1, dtype=np.int32)
    case.table = np.concatenate([case.table, extra], axis=1)


@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ctx,trees,hq,hkv,d,pt", [
    ([0, 1, 63, 64, 65, 127, 128, 129], [1, 3, 2, 5, 1, 9, 8, 9], 4, 2, 128, 16),   # 18 rows, around a step
    ([37, 300, 0], [8, 0, 4], 32, 8, 128, 16),
    ([129, 700], [13, 7], 16, 2, 64, 8),
    ([1000], [33], 8, 8, 128, 16),
    ([250, 90], [24, 17], 8, 4, 96, 24),
    ([130], [6], 9, 3, 16, 32),
    ([0], [64], 1, 1, 40, 16),
    ([5000, 3], [4, 20], 6, 2, 128, 256),                                           # pages of two steps
])
def test_plan_for_long_contexts(kv, name, ctx, trees, hq, hkv, d, pt):
    torch = torch_cuda()
    if kv != "f16" and d % 16:
        d = 48
    case = Case(torch, np.random.default_rng(sum(ctx) + hq + d), ctx, trees, hq, hkv, d, pt, kv, name)
    _widen_table(case, MANY)
    case.check(case.run(max_ctx=MANY))


@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
@pytest.mark.parametrize("max_ctx", [1, 70, MANY])
def test_contexts_past_the_bound(kv, max_ctx):
    """max_ctx sizes the plan; lengths above it cost time, not results."""
    torch = torch_cuda()
    for trees in ([3, 2], [20, 9]):
        case = Case(torch, np.random.default_rng(91), [900, 130], trees, 8, 2, 128, 16, kv, "f32")
        _widen_table(case, max_ctx)
        case.check(case.run(max_ctx=max_ctx))


@pytest.mark.parametrize("kv", ["f16", "fp8", "int8"])
def test_single_long_context_few_rows(kv):
    """More context pieces than a warp has lanes."""
    torch = torch_cuda()
    case = Case(torch, np.random.default_rng(93), [9001], [2], 4, 1, 128, 16, kv, "f32")
    case.check(case.run())
