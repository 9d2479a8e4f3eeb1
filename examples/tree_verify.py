"""One round of speculative verification on a small random-init model.

A draft proposes a tree of tokens per sequence; one pass of the model scores
every node, the longest path that the model itself would have taken is
committed, and the pass's next token comes for free.  A layer is

    int4 q/k/v projection with RMSNorm -> rotary positions (by depth in the tree)
    -> 8-bit KV append -> tree attention over the pages -> int4 output projection

and the tree's children are scored with log probabilities from the logits.  The
result is checked against decoding token by token.

    python examples/tree_verify.py            # needs a B200 and the built library
"""
import ctypes
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "vspec-engine_b200", "python"))
import vspec_b200 as V  # noqa: E402

LAYERS, HIDDEN, HQ, HKV, D, VOCAB = 2, 512, 8, 2, 64, 4096
PAGE, MAX_PAGES = 16, 12
QKV = (HQ + 2 * HKV) * D
BLOCK = 128


class Linear:
    """int4 weights, quantised and packed on the device."""

    def __init__(self, n, k, gen):
        w = torch.randn((n, k), device="cuda", generator=gen) / k ** 0.5
        self.n, self.k, self.groups = n, k, k // BLOCK
        self.packed = torch.empty((n, k // 2), dtype=torch.uint8, device="cuda")
        self.scales, self.zp = (torch.empty((n, self.groups), device="cuda") for _ in range(2))
        V.check(V.lib.vspec_b200_quantize_rowwise(w.data_ptr(), n, k, 4, BLOCK, ctypes.c_double(1.0),
                                                  self.packed.data_ptr(), self.scales.data_ptr(), self.zp.data_ptr(),
                                                  None), "quantize_rowwise")

    def __call__(self, x, norm=None, residual=None):
        y = torch.empty((x.shape[0], self.n), device="cuda")
        V.lowbit_linear(x.data_ptr(), self.packed.data_ptr(), self.scales.data_ptr(), self.zp.data_ptr(), y.data_ptr(),
                        x.shape[0], self.n, self.k, self.groups, 4,
                        flags=(V.F_RMSNORM if norm is not None else 0) | (V.F_RESIDUAL if residual is not None else 0),
                        norm_weight=norm.data_ptr() if norm is not None else None,
                        residual=residual.data_ptr() if residual is not None else None)
        return y


class Cache:
    """fp8 pages of one layer: codes and one scale per row, K and V."""

    def __init__(self, pages):
        self.codes = [torch.zeros((pages * PAGE, HKV, D), dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.scales = [torch.zeros((pages * PAGE, HKV), device="cuda") for _ in range(2)]
        self.pages = pages

    def copy(self):
        c = Cache(self.pages)
        for dst, src in zip(c.codes + c.scales, self.codes + self.scales):
            dst.copy_(src)
        return c

    def ptrs(self):
        return [t.data_ptr() for t in self.codes + self.scales]

    def append(self, k, v, k_stride, v_stride, slots):
        kc, vc, ks, vs = self.ptrs()
        V.kv_quant_append(k, v, slots.data_ptr(), slots.numel(), HKV, D, self.pages * PAGE, V.KV_FP8, kc, vc, ks, vs,
                          k_stride=k_stride, v_stride=v_stride)

    def rows(self, table, lens):
        """The first tokens of every sequence as fp16 rows, e.g. for a store of prefixes."""
        total = int(sum(lens))
        cu = ints([0] + list(np.cumsum(lens)))
        out = [torch.empty((total, HKV, D), dtype=torch.float16, device="cuda") for _ in range(2)]
        V.kv_quant_gather(*self.ptrs(), table.data_ptr(), cu.data_ptr(), len(lens), total, HKV, D, PAGE, MAX_PAGES,
                          self.pages, V.KV_FP8, out[0].data_ptr(), out[1].data_ptr())
        return out


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


class Model:
    def __init__(self, seed):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        self.embed = torch.randn((VOCAB, HIDDEN), device="cuda", generator=gen)
        self.qkv = [Linear(QKV, HIDDEN, gen) for _ in range(LAYERS)]
        self.out = [Linear(HIDDEN, HQ * D, gen) for _ in range(LAYERS)]
        self.norm = torch.ones(HIDDEN, device="cuda")
        self.head = Linear(VOCAB, HIDDEN, gen)
        turns, self.rope_factor = V.rope_turns(D, 10000.0)
        self.turns = torch.from_numpy(turns.view(np.int64)).cuda()

    def __call__(self, caches, tokens, pos, slots, table, ctx, trees, mask=None):
        """Logits [rows][VOCAB] of the rows of all sequences' trees, and the K and V rows of each layer."""
        rows, words = len(tokens), 0 if mask is None else mask.shape[1]
        pos, slots, ctx_d, cu = ints(pos), ints(slots), ints(ctx), ints([0] + list(np.cumsum(trees)))
        mask_d = None if mask is None else torch.from_numpy(mask.view(np.int32).copy()).cuda()
        x = self.embed[torch.as_tensor(tokens, device="cuda")]
        kept = []
        for layer, cache in enumerate(caches):
            y = self.qkv[layer](x, norm=self.norm)
            q, k, v = (y.data_ptr() + 4 * o for o in (0, HQ * D, (HQ + HKV) * D))
            V.rope(q, k, q, k, pos.data_ptr(), self.turns.data_ptr(), rows, HQ, HKV, D, D, attn_factor=self.rope_factor,
                   q_stride=QKV, k_stride=QKV, q_out_stride=QKV, k_out_stride=QKV)
            cache.append(k, v, QKV, QKV, slots)
            a = torch.empty((rows, HQ * D), device="cuda")
            kc, vc, ks, vs = cache.ptrs()
            V.tree_attention(q, kc, vc, ks, vs, table.data_ptr(), ctx_d.data_ptr(), cu.data_ptr(),
                             None if mask is None else mask_d.data_ptr(), a.data_ptr(), len(trees), rows, max(trees),
                             HQ, HKV, D, PAGE, MAX_PAGES, cache.pages, MAX_PAGES * PAGE, D ** -0.5, kv_dtype=V.KV_FP8,
                             mask_words=words, q_stride=QKV)
            x = self.out[layer](a, residual=x)
            kept.append(y)
        return self.head(x, norm=self.norm), kept


def score(logits, given, top_k):
    """log p of `given` [rows][n] (-1: none), the entropies, and the best alternatives of every row."""
    rows, n = given.shape
    g = ints(given)
    lp, ent = torch.empty((rows, n), device="cuda"), torch.empty(rows, device="cuda")
    top, ids = torch.empty((rows, top_k), device="cuda"), torch.empty((rows, top_k), dtype=torch.int32, device="cuda")
    V.logprobs(logits.data_ptr(), rows, VOCAB, tokens=g.data_ptr(), num_tokens=n, token_logprobs=lp.data_ptr(),
               entropy=ent.data_ptr(), top_k=top_k, top_logprobs=top.data_ptr(), top_ids=ids.data_ptr())
    torch.cuda.synchronize()
    return lp.cpu().numpy(), ent.cpu().numpy(), top.cpu().numpy(), ids.cpu().numpy()


# node -> parent; nodes 1, 3, 5 are what the model would say, the others a wrong guess
PARENT = [-1, 0, 0, 1, 1, 3, 3, 2]
RIGHT = [1, 3, 5]


def main(seed=0):
    rng = np.random.default_rng(seed)
    model = Model(seed)
    prompts = [rng.integers(0, VOCAB, n) for n in (37, 90)]
    batch, ctx = len(prompts), [0, 0]
    perm = rng.permutation(batch * MAX_PAGES).astype(np.int32).reshape(batch, MAX_PAGES)
    table = torch.from_numpy(perm).cuda()
    slot = lambda b, t: int(perm[b, t // PAGE]) * PAGE + t % PAGE   # noqa: E731
    caches = [Cache(batch * MAX_PAGES) for _ in range(LAYERS)]

    # prompts: a chain each, one call for both
    lens = [len(p) for p in prompts]
    at = [(b, t) for b in range(batch) for t in range(lens[b])]
    logits, _ = model(caches, np.concatenate(prompts), [t for _, t in at], [slot(b, t) for b, t in at], table, ctx, lens)
    last = logits[torch.as_tensor(np.cumsum(lens) - 1, device="cuda")].contiguous()
    root = score(last, np.full((batch, 1), -1), 1)[3][:, 0]
    ctx = lens

    # token by token: what the tree has to agree with
    plain = [c.copy() for c in caches]
    said, said_lp, now = [root], [], root
    for i in range(len(RIGHT) + 1):
        pos = [c + i for c in ctx]
        logits, _ = model(plain, now, pos, [slot(b, t) for b, t in enumerate(pos)], table, pos, [1] * batch)
        _, _, top, ids = score(logits, np.full((batch, 1), -1), 1)
        now = ids[:, 0]
        said.append(now)
        said_lp.append(top[:, 0])

    # the draft: right tokens on one path, wrong ones beside it
    nodes = len(PARENT)
    depth = [0] * nodes
    bits = np.zeros((nodes, 1), dtype=np.uint32)
    for j, parent in enumerate(PARENT):
        if parent >= 0:
            depth[j] = depth[parent] + 1
            bits[j] = bits[parent]
        bits[j, 0] |= np.uint32(1 << j)
    draft = np.zeros((batch, nodes), dtype=np.int64)
    for b in range(batch):
        for j in range(nodes):
            right = said[depth[j]][b]
            draft[b, j] = right if j == 0 or j in RIGHT else (right + 1 + j) % VOCAB
    at = [(b, j) for b in range(batch) for j in range(nodes)]
    logits, kept = model(caches, draft.reshape(-1), [ctx[b] + depth[j] for b, j in at],
                         [slot(b, ctx[b] + j) for b, j in at], table, ctx, [nodes] * batch, np.tile(bits, (batch, 1)))
    children = [[c for c in range(nodes) if PARENT[c] == j] for j in range(nodes)]
    given = np.full((batch * nodes, 2), -1)
    for b, j in at:
        given[b * nodes + j, :len(children[j])] = draft[b, children[j]]
    lp, _, top, ids = score(logits, given, 5)

    # walk from the root while the model's own choice is among the children
    paths, worst = [], 0.0
    for b in range(batch):
        path = [0]
        while True:
            r = b * nodes + path[-1]
            worst = max(worst, abs(float(top[r, 0]) - float(said_lp[len(path) - 1][b])))
            hit = [i for i, c in enumerate(children[path[-1]]) if draft[b, c] == ids[r, 0]]
            if not hit:
                break
            assert lp[r, hit[0]] == top[r, 0]
            path.append(children[path[-1]][hit[0]])
        assert path == [0] + RIGHT and ids[b * nodes + path[-1], 0] == said[-1][b]
        paths.append(path)

    # commit: the accepted rows move to the places behind the context
    src = torch.as_tensor([b * nodes + j for b in range(batch) for j in paths[b]], device="cuda")
    slots = ints([slot(b, ctx[b] + i) for b in range(batch) for i in range(len(paths[b]))])
    for cache, y in zip(caches, kept):
        rows = y[src]
        cache.append(rows.data_ptr() + 4 * HQ * D, rows.data_ptr() + 4 * (HQ + HKV) * D, QKV, QKV, slots)
    ctx = [c + len(p) for c, p in zip(ctx, paths)]
    drift = 0.0
    for cache, other in zip(caches, plain):
        for a, b in zip(cache.rows(table, ctx), other.rows(table, ctx)):
            drift = max(drift, ((a.float() - b.float()).abs().max() / b.float().abs().max()).item())
    assert V.page_fault_flag() == 0 and V.tree_attention_timeout_flag() == 0
    print(f"accepted {[len(p) - 1 for p in paths]} drafted tokens and one more each in one pass; against token by "
          f"token: log probabilities within {worst:.1e}, committed cache within {drift:.1e}")
    return worst, drift


if __name__ == "__main__":
    main()
