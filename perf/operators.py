"""The operators of a speculative verification step, as a serving program calls them.

A step checks a tree of drafted tokens for every sequence of a batch at once.  Five calls make it up:

  rope         rotary positions of the fused q/k/v projection's q and k rows (a drafted token's position is
               its depth in the tree, not its row)
  kv_append    the new K and V rows, quantised to e4m3 or int8 codes with one scale a row and head, into pages
  kv_gather    pages read back: the K and V rows of whole sequences as plain tensors
  tree         attention of the drafted tokens over their sequence's pages, each seeing the prefix and the
               drafted tokens that its mask names
  logprobs     log probabilities of the drafted children, entropy and the best alternatives from the logits

`run` computes them in plain torch, or, where `own` is true, through the library's binding.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TWO_PI = 2.0 * math.pi
_FP8_MAX, _INT8_MAX = 448.0, 127.0

# The largest listed case of each operator, as the product that draw() keeps its cases under.
_ROPE_MOST = 8192 * 40 * 128
_KV_MOST = 16384 * 8 * 128
_TREE_MOST = 32 * 64 * 32 * 128 * 4352
_LOGITS_MOST = 512 * 151936


def listed():
    return [
        # one sequence's eight drafted tokens: launch latency is all there is
        dict(name="rope_verify8", op="rope", tokens=8, hq=32, hk=8, d=128, rot=128, dtype="f32", inter=False,
             scaling="plain", max_pos=4096),
        # a prompt in 16-bit, interleaved pairs, half of the head rotated, positions stretched eightfold
        dict(name="rope_prompt8192", op="rope", tokens=8192, hq=32, hk=8, d=128, rot=64, dtype="bf16", inter=True,
             scaling="yarn", max_pos=131072),
        # 32 sequences x 16 drafted tokens appended in e4m3
        dict(name="kv_append_512_fp8", op="kv_append", rows=512, heads=8, d=128, dtype="f32", kv="fp8"),
        # a chunk of prompts appended in int8, 16-bit source rows
        dict(name="kv_append_16384_int8", op="kv_append", rows=16384, heads=8, d=128, dtype="f16", kv="int8"),
        # one cached prefix of odd length read back, scattered pages
        dict(name="kv_gather_1x777_int8", op="kv_gather", batch=1, lo=777, hi=777, heads=8, d=128, pt=16, kv="int8",
             dtype="f32"),
        # eight long prefixes read back in 16-bit for a prompt's attention
        dict(name="kv_gather_8x2048_fp8", op="kv_gather", batch=8, lo=512, hi=3584, heads=8, d=128, pt=16, kv="fp8",
             dtype="f16"),
        # one sequence, a small tree: the latency of a single user's step
        dict(name="tree_1x8_ctx768", op="tree", batch=1, q=8, hq=32, hkv=8, d=128, lo=768, hi=768, pt=16, kv="f16",
             dtype="f32", ragged=False),
        # 8 sequences with 16 drafted tokens over e4m3 pages, contexts of a few thousand
        dict(name="tree_8x16_fp8", op="tree", batch=8, q=16, hq=32, hkv=8, d=128, lo=1024, hi=6144, pt=16, kv="fp8",
             dtype="f16", ragged=False),
        # trees of uneven size, an empty one and an empty context among them, eight query heads a KV head, int8
        dict(name="tree_5x13_ragged_int8", op="tree", batch=5, q=13, hq=64, hkv=8, d=128, lo=333, hi=2077, pt=16,
             kv="int8", dtype="bf16", ragged=True),
        # a full batch with wide trees: the most arithmetic a step has
        dict(name="tree_32x64_ctx8192", op="tree", batch=32, q=64, hq=32, hkv=8, d=128, lo=512, hi=8192, pt=16,
             kv="f16", dtype="f32", ragged=False),
        # one sequence's tree, five alternatives wanted
        dict(name="logprobs_8_f32", op="logprobs", rows=8, vocab=151936, dtype="f32", given=3, top=5, allowed=False),
        # 32 sequences x 16 drafted tokens, twenty alternatives
        dict(name="logprobs_512_f32", op="logprobs", rows=512, vocab=151936, dtype="f32", given=4, top=20,
             allowed=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "kv_append", "kv_gather", "tree", "tree", "logprobs"])
    heads = [(32, 8), (64, 8), (8, 8), (16, 2), (4, 1)]
    if op == "rope":
        hq, hk = rng.choice(heads)
        d = rng.choice([64, 80, 128, 128, 256])
        rot = rng.choice([d, d, d // 2, d // 4])
        tokens = min(_log_int(rng, 1, 8192), _ROPE_MOST // ((hq + hk) * d))
        return dict(op=op, tokens=tokens, hq=hq, hk=hk, d=d, rot=rot, dtype=rng.choice(list(_TYPES)),
                    inter=rng.random() < 0.5, scaling=rng.choice(["plain", "linear", "ntk", "yarn"]),
                    max_pos=_log_int(rng, 256, 1 << 20))
    if op == "kv_append":
        h, d = rng.choice([8, 8, 2, 5, 16]), rng.choice([64, 128, 128, 256])
        rows = min(_log_int(rng, 1, 16384), _KV_MOST // (h * d))
        return dict(op=op, rows=rows, heads=h, d=d, dtype=rng.choice(list(_TYPES)), kv=rng.choice(["fp8", "int8"]))
    if op == "kv_gather":
        h, d = rng.choice([8, 8, 2, 5, 16]), rng.choice([64, 128, 128, 256])
        batch = _log_int(rng, 1, 32)
        hi = max(1, min(_log_int(rng, 16, 16384), _KV_MOST // (h * d * batch)))
        return dict(op=op, batch=batch, lo=rng.randint(0, hi), hi=hi, heads=h, d=d, pt=rng.choice([16, 16, 32, 5]),
                    kv=rng.choice(["fp8", "int8"]), dtype=rng.choice(list(_TYPES)))
    if op == "tree":
        hq, hkv = rng.choice(heads)
        d = rng.choice([64, 128, 128, 96])
        batch, q = _log_int(rng, 1, 32), _log_int(rng, 1, 64)
        hi = max(1, min(_log_int(rng, 16, 32768), _TREE_MOST // (batch * q * hq * d)))
        return dict(op=op, batch=batch, q=q, hq=hq, hkv=hkv, d=d, lo=rng.randint(hi // 4, hi), hi=hi,
                    pt=rng.choice([16, 16, 16, 64, 24]), kv=rng.choice(["f16", "fp8", "int8"]),
                    dtype=rng.choice(list(_TYPES)), ragged=rng.random() < 0.5)
    vocab = rng.choice([1000, 32000, 65537, 151936])
    return dict(op=op, rows=max(1, min(_log_int(rng, 1, 1024), _LOGITS_MOST // vocab)), vocab=vocab,
                dtype=rng.choice(list(_TYPES)), given=rng.randint(1, 8), top=rng.randint(1, 32),
                allowed=rng.random() < 0.3)


# ------------------------------------------------------------------------------------------------ sizes of a case

def _lengths(case):
    """Cached tokens of each sequence: spread over [lo, hi], in no order."""
    n = case["batch"]
    if n == 1:
        return [case["hi"]]
    step = next(s for s in (37, 41, 43, 47) if math.gcd(s, n) == 1)
    got = [case["lo"] + (case["hi"] - case["lo"]) * ((i * step) % n) // (n - 1) for i in range(n)]
    if case.get("ragged") and n > 2:
        got[2] = 0
    return got


def _drafted(case):
    """Drafted tokens of each sequence."""
    n, q = case["batch"], case["q"]
    if not case["ragged"]:
        return [q] * n
    return [0 if i == 1 else q - (i * 5) % q for i in range(n)]


def _bytes_of(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    op = case["op"]
    if op == "rope":
        elems = case["tokens"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * elems * _bytes_of(case["dtype"]) + 4 * case["tokens"],
                "flops": 3 * elems * case["rot"] / case["d"]}
    if op == "kv_append":
        rows = case["rows"] * case["heads"]
        return {"bytes": 2 * rows * (case["d"] * (_bytes_of(case["dtype"]) + 1) + 4) + 4 * case["rows"],
                "flops": 2 * rows * case["d"] * 3}
    if op == "kv_gather":
        rows = sum(_lengths(case)) * case["heads"]
        return {"bytes": 2 * rows * (case["d"] * (_bytes_of(case["dtype"]) + 1) + 4), "flops": 2 * rows * case["d"]}
    if op == "tree":
        ctx, t = _lengths(case), _drafted(case)
        cached = sum(c + n for c, n in zip(ctx, t) if n) * case["hkv"]
        kv = cached * case["d"] * 2 * (2 if case["kv"] == "f16" else 1) + (0 if case["kv"] == "f16" else cached * 8)
        io = 2 * sum(t) * case["hq"] * case["d"] * _bytes_of(case["dtype"])
        return {"bytes": kv + io, "flops": 4 * case["d"] * case["hq"] * sum(n * (c + n / 2) for c, n in zip(ctx, t))}
    n = case["rows"] * case["vocab"]
    out = case["rows"] * (4 * case["given"] * 2 + 4 + 8 * case["top"])
    return {"bytes": n * _bytes_of(case["dtype"]) + (n / 8 if case["allowed"] else 0) + out, "flops": 6 * n}


# ------------------------------------------------------------------------------------------------------- inputs

def _rope_freqs(case, theta=1e6, factor=8.0, original=4096, fast=32.0, slow=1.0):
    """Turns a position adds to each pair's angle, as fractions of 2^64, and the factor on cos and sin."""
    rot, scaling = case["rot"], case["scaling"]
    i = np.arange(rot // 2, dtype=np.float64)
    if scaling == "ntk":
        theta = theta * factor ** (rot / max(rot - 2, 1))
    f = theta ** (-2.0 * i / rot)
    mult = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        where = [rot * math.log(original / (b * _TWO_PI)) / (2.0 * math.log(theta)) for b in (fast, slow)]
        lo, hi = max(math.floor(where[0]), 0), min(math.ceil(where[1]), rot - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        f = f * (1.0 - ramp) + f / factor * ramp
        mult = 0.1 * math.log(factor) + 1.0
    return (f / _TWO_PI * 2.0 ** 64).astype(np.uint64), mult


def _quantise(x, kv):
    """Codes and scales of rows [..., d], M the largest code: scale = absmax / M, code = x * (M / absmax) to nearest
    even."""
    most = torch.full((), _FP8_MAX if kv == "fp8" else _INT8_MAX, device=x.device)
    x = x.float()
    top = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().amax(-1)
    scale, c = top / most, x * (most / top).unsqueeze(-1)
    c = torch.where(torch.isnan(c), torch.zeros_like(c), c).clamp(-most, most)
    return (c.to(torch.float8_e4m3fn) if kv == "fp8" else c.round().to(torch.int8)), scale


def _pages(g, dev, lengths, pt, spare=3):
    """Page table [batch][most pages] of a random permutation of the pool, and the pool's page count."""
    need = [-(-n // pt) for n in lengths]
    total, most = sum(need) + spare, max(max(need), 1)
    perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((len(lengths), most), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    st = dict(case)
    op = case["op"]
    dt = _TYPES.get(case["dtype"])
    if op == "rope":
        t, hq, hk, d = case["tokens"], case["hq"], case["hk"], case["d"]
        turns, mult = _rope_freqs(case)
        qkv = normal(t, (hq + 2 * hk) * d).to(dt)
        st.update(qkv=qkv, q=qkv[:, :hq * d], k=qkv[:, hq * d:(hq + hk) * d], mult=mult,
                  pos=torch.randint(0, case["max_pos"], (t,), generator=g, device=dev, dtype=torch.int32),
                  turns=torch.from_numpy(turns.view(np.int64)).to(dev),
                  q_out=torch.empty((t, hq, d), dtype=dt, device=dev),
                  k_out=torch.empty((t, hk, d), dtype=dt, device=dev))
    elif op == "kv_append":
        r, h, d = case["rows"], case["heads"], case["d"]
        pool = r + 37
        kv = normal(r, 2 * h * d)
        # projections have a few channels far larger than the rest
        kv[:, torch.randint(0, 2 * h * d, (h,), generator=g, device=dev)] *= 12.0
        kv = kv.to(dt)
        codes = torch.float8_e4m3fn if case["kv"] == "fp8" else torch.int8
        st.update(src=kv, k=kv[:, :h * d], v=kv[:, h * d:], pool=pool,
                  slots=torch.randperm(pool, generator=g, device=dev)[:r].to(torch.int32),
                  k_codes=torch.zeros((pool, h, d), dtype=torch.uint8, device=dev).view(codes),
                  v_codes=torch.zeros((pool, h, d), dtype=torch.uint8, device=dev).view(codes),
                  k_scales=torch.zeros((pool, h), device=dev), v_scales=torch.zeros((pool, h), device=dev))
    elif op == "kv_gather":
        h, d, pt = case["heads"], case["d"], case["pt"]
        lens = _lengths(case)
        table, pages = _pages(g, dev, lens, pt)
        for n in "kv":
            st[n + "_codes"], st[n + "_scales"] = _quantise(normal(pages * pt, h, d), case["kv"])
        total = sum(lens)
        seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
        at = torch.cat([torch.arange(n) for n in lens])
        st.update(table=table, pages=pages, total=total, seq=seq.to(dev), at=at.to(dev),
                  cu=torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=dev),
                  k_out=torch.empty((total, h, d), dtype=dt, device=dev),
                  v_out=torch.empty((total, h, d), dtype=dt, device=dev))
    elif op == "tree":
        hq, hkv, d, pt, q = case["hq"], case["hkv"], case["d"], case["pt"], case["q"]
        lens, trees = _lengths(case), _drafted(case)
        table, pages = _pages(g, dev, [c + n for c, n in zip(lens, trees)], pt)
        for n in "kv":
            x = normal(pages * pt, hkv, d)
            if case["kv"] == "f16":
                st[n + "_codes"], st[n + "_scales"] = x.half(), None
            else:
                st[n + "_codes"], st[n + "_scales"] = _quantise(x, case["kv"])
        total, words = sum(trees), -(-q // 32)
        r = random.Random(seed)
        bits = np.zeros((total, words), dtype=np.uint32)
        row = 0
        for b, n in enumerate(trees):
            for j in range(n):
                parent = r.randint(-1, j - 1)
                if parent >= 0:
                    bits[row + j] = bits[row + parent]
                bits[row + j, j // 32] |= np.uint32(1 << (j % 32))
            if lens[b] == 0 and n > 1:
                bits[row + n - 1] = 0  # a row that sees nothing
            row += n
        st.update(table=table, pages=pages, total=total, words=words, max_ctx=max(c + n for c, n in zip(lens, trees)),
                  qs=normal(total, hq, d).to(dt), mask=torch.from_numpy(bits.view(np.int32)).to(dev),
                  ctx=torch.tensor(lens, dtype=torch.int32, device=dev),
                  cu=torch.tensor([0] + list(np.cumsum(trees)), dtype=torch.int32, device=dev),
                  padded=torch.tensor([b * q + j for b, n in enumerate(trees) for j in range(n)], device=dev),
                  scale=1.0 / math.sqrt(d), out=torch.empty((total, hq, d), dtype=dt, device=dev))
    else:
        rows, v = case["rows"], case["vocab"]
        x = normal(rows, v) * 2.5
        best = torch.randint(0, v, (rows, 4), generator=g, device=dev)
        x.scatter_add_(1, best, torch.full((rows, 4), 12.0, device=dev))
        st.update(logits=x.to(dt), mask=None,
                  tokens=torch.randint(0, v, (rows, case["given"]), generator=g, device=dev, dtype=torch.int32),
                  token_lp=torch.empty((rows, case["given"]), device=dev), entropy=torch.empty((rows,), device=dev),
                  top_lp=torch.empty((rows, case["top"]), device=dev),
                  top_ids=torch.empty((rows, case["top"]), dtype=torch.int32, device=dev), inv_t=1.0 / 0.8)
        st["tokens"][:, 0] = best[:, 0]
        if case["allowed"]:
            st["mask"] = torch.randint(-(1 << 31), 1 << 31, (rows, -(-v // 32)), generator=g, device=dev,
                                       dtype=torch.int64).to(torch.int32)
    return st


# ---------------------------------------------------------------------------------------------------- plain form

def _rope_plain(s, x, heads):
    d, rot = s["d"], s["rot"]
    x = x.reshape(-1, heads, d).float()
    # position x turns as a 64-bit fraction of a turn: the product's overflow drops whole turns
    part = (s["pos"].long().unsqueeze(1) * s["turns"]) >> 32
    angle = part.float() * (_TWO_PI / 2.0 ** 32)
    cos, sin = (torch.cos(angle) * s["mult"]).unsqueeze(1), (torch.sin(angle) * s["mult"]).unsqueeze(1)
    if s["inter"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    return torch.cat([y, x[..., rot:]], dim=-1).to(s["q_out"].dtype)


def _kv_append_plain(s):
    at = s["slots"].long()
    for n in "kv":
        codes, scales = _quantise(s[n].reshape(-1, s["heads"], s["d"]), s["kv"])
        s[n + "_codes"].view(torch.uint8)[at] = codes.view(torch.uint8)
        s[n + "_scales"][at] = scales
    return [s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]]


def _kv_gather_plain(s):
    slot = s["table"][s["seq"], s["at"] // s["pt"]].long() * s["pt"] + s["at"] % s["pt"]
    got = []
    for n in "kv":
        c = s[n + "_codes"].view(torch.uint8)[slot].view(s[n + "_codes"].dtype).float()
        got.append((c * s[n + "_scales"][slot].unsqueeze(-1)).to(s["k_out"].dtype))
    return got


def _tree_plain(s):
    batch, t, hq, hkv, d, pt = s["batch"], s["q"], s["hq"], s["hkv"], s["d"], s["pt"]
    span = s["table"].shape[1] * pt
    kv = []
    for n in "kv":
        x = s[n + "_codes"]
        x = (x if s["kv"] == "f16" else x.view(torch.uint8)).view(-1, pt, hkv, d)[s["table"].long()]
        x = x.view(s[n + "_codes"].dtype).float().view(batch, span, hkv, d)
        if s["kv"] != "f16":
            x = x * s[n + "_scales"].view(-1, pt, hkv)[s["table"].long()].view(batch, span, hkv, 1)
        kv.append(x.transpose(1, 2))
    q = torch.zeros((batch * t, hq, d), device=s["qs"].device)
    q[s["padded"]] = s["qs"].float()
    q = q.view(batch, t, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, d)
    seen = torch.zeros((batch * t, s["words"] * 32), dtype=torch.bool, device=q.device)
    seen[s["padded"]] = ((s["mask"].unsqueeze(-1) >> torch.arange(32, device=q.device)) & 1).bool().flatten(1)
    seen = seen.view(batch, t, -1)
    at = torch.arange(span, device=q.device)
    drafted = at.unsqueeze(0) - s["ctx"].long().unsqueeze(1)  # place among the drafted tokens, below 0: prefix
    inside = (drafted >= 0) & (drafted < t)
    look = torch.gather(seen, 2, drafted.clamp(0, t - 1).unsqueeze(1).expand(-1, t, -1))
    look = (drafted < 0).unsqueeze(1) | (look & inside.unsqueeze(1))  # [batch][t][span]
    look = look.unsqueeze(1).expand(-1, hq // hkv, -1, -1).reshape(batch, 1, -1, span)
    score = torch.matmul(q, kv[0].transpose(2, 3)) * s["scale"]
    score = torch.where(look, score, torch.full((), -math.inf, device=q.device))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, kv[1]) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.view(batch, hkv, hq // hkv, t, d).permute(0, 3, 1, 2, 4).reshape(batch * t, hq, d)
    return out[s["padded"]].to(s["out"].dtype)


def _logprobs_plain(s):
    raw = s["logits"]
    x = raw.float() * s["inv_t"]
    if s["mask"] is not None:
        bit = torch.arange(32, device=x.device)
        ok = ((s["mask"].unsqueeze(-1) >> bit) & 1).bool().flatten(1)[:, :s["vocab"]]
        x = torch.where(ok, x, torch.full((), -math.inf, device=x.device))
        raw = torch.where(ok, raw, torch.full((), -math.inf, device=x.device, dtype=raw.dtype))
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    weighted = torch.where(e > 0, e * (x - m), torch.zeros_like(e)).sum(-1, keepdim=True)
    entropy = torch.log(total) - weighted / total
    ids = torch.sort(raw, dim=-1, descending=True, stable=True).indices[:, :s["top"]]
    return [torch.gather(x, 1, s["tokens"].long()) - lse, entropy.squeeze(1), torch.gather(x, 1, ids) - lse,
            ids.to(torch.int32)]


# ------------------------------------------------------------------------------------------------- the library's

_binding = None


def _lib():
    global _binding
    if _binding is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "vspec-engine_b200", "python"))
        import vspec_b200
        _binding = vspec_b200
    return _binding


def _run_own(s):
    V = _lib()
    types = {"f32": V.T_F32, "f16": V.T_F16, "bf16": V.T_BF16}
    kinds = {"f16": V.KV_F16, "fp8": V.KV_FP8, "int8": V.KV_INT8}
    stream = torch.cuda.current_stream().cuda_stream
    op = s["op"]
    if op == "rope":
        V.rope(s["q"].data_ptr(), s["k"].data_ptr(), s["q_out"].data_ptr(), s["k_out"].data_ptr(), s["pos"].data_ptr(),
               s["turns"].data_ptr(), s["tokens"], s["hq"], s["hk"], s["d"], s["rot"], types[s["dtype"]],
               interleaved=s["inter"], attn_factor=s["mult"], q_stride=s["qkv"].shape[1], k_stride=s["qkv"].shape[1],
               stream=stream)
        return [s["q_out"], s["k_out"]]
    if op == "kv_append":
        V.kv_quant_append(s["k"].data_ptr(), s["v"].data_ptr(), s["slots"].data_ptr(), s["rows"], s["heads"], s["d"],
                          s["pool"], kinds[s["kv"]], s["k_codes"].data_ptr(), s["v_codes"].data_ptr(),
                          s["k_scales"].data_ptr(), s["v_scales"].data_ptr(), src_dtype=types[s["dtype"]],
                          k_stride=s["src"].shape[1], v_stride=s["src"].shape[1], stream=stream)
        return [s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"]]
    if op == "kv_gather":
        V.kv_quant_gather(s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scales"].data_ptr(),
                          s["v_scales"].data_ptr(), s["table"].data_ptr(), s["cu"].data_ptr(), s["batch"], s["total"],
                          s["heads"], s["d"], s["pt"], s["table"].shape[1], s["pages"], kinds[s["kv"]],
                          s["k_out"].data_ptr(), s["v_out"].data_ptr(), out_dtype=types[s["dtype"]], stream=stream)
        return [s["k_out"], s["v_out"]]
    if op == "tree":
        quantised = s["kv"] != "f16"
        V.tree_attention(s["qs"].data_ptr(), s["k_codes"].data_ptr(), s["v_codes"].data_ptr(),
                         s["k_scales"].data_ptr() if quantised else None,
                         s["v_scales"].data_ptr() if quantised else None, s["table"].data_ptr(), s["ctx"].data_ptr(),
                         s["cu"].data_ptr(), s["mask"].data_ptr(), s["out"].data_ptr(), s["batch"], s["total"], s["q"],
                         s["hq"], s["hkv"], s["d"], s["pt"], s["table"].shape[1], s["pages"], s["max_ctx"], s["scale"],
                         q_dtype=types[s["dtype"]], kv_dtype=kinds[s["kv"]], mask_words=s["words"], stream=stream)
        return s["out"]
    V.logprobs(s["logits"].data_ptr(), s["rows"], s["vocab"], types[s["dtype"]], tokens=s["tokens"].data_ptr(),
               num_tokens=s["given"], token_logprobs=s["token_lp"].data_ptr(), entropy=s["entropy"].data_ptr(),
               top_k=s["top"], top_logprobs=s["top_lp"].data_ptr(), top_ids=s["top_ids"].data_ptr(),
               allowed=s["mask"].data_ptr() if s["mask"] is not None else None, inv_temperature=s["inv_t"],
               stream=stream)
    return [s["token_lp"], s["entropy"], s["top_lp"], s["top_ids"]]


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "rope":
        return [_rope_plain(state, state["q"], state["hq"]), _rope_plain(state, state["k"], state["hk"])]
    if op == "kv_append":
        return _kv_append_plain(state)
    if op == "kv_gather":
        return _kv_gather_plain(state)
    if op == "tree":
        return _tree_plain(state)
    return _logprobs_plain(state)


# ------------------------------------------------------------------------------------------------ in 64 bits

def _exact_rope(s):
    f = s["turns"].cpu().numpy().view(np.uint64).astype(np.float64) / 2.0 ** 64  # turns a position
    whole = np.outer(s["pos"].cpu().numpy().astype(np.float64), f)
    angle = torch.from_numpy((whole - np.rint(whole)) * _TWO_PI).to(s["q"].device)
    turn = torch.polar(torch.full_like(angle, s["mult"]), angle).unsqueeze(1)
    got = []
    for x, h in ((s["q"], s["hq"]), (s["k"], s["hk"])):
        x = x.reshape(-1, h, s["d"]).double()
        half, rot = s["rot"] // 2, s["rot"]
        first = x[..., 0:rot:2] if s["inter"] else x[..., :half]
        second = x[..., 1:rot:2] if s["inter"] else x[..., half:rot]
        z = torch.complex(first.contiguous(), second.contiguous()) * turn
        y = x.clone()
        if s["inter"]:
            y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
        else:
            y[..., :half], y[..., half:rot] = z.real, z.imag
        got.append(y)
    return got


def _exact_kv_append(s):
    got = []
    most = _FP8_MAX if s["kv"] == "fp8" else _INT8_MAX
    for n in "kv":
        x = s[n].reshape(-1, s["heads"], s["d"]).double()
        scale = x.abs().max(dim=-1).values / most
        pool = torch.zeros((s["pool"], s["heads"]), dtype=torch.float64, device=x.device)
        pool[s["slots"].long()] = scale
        codes = None  # an int8 code is a whole number
        if s["kv"] == "fp8":
            codes = torch.zeros((s["pool"], s["heads"], s["d"]), dtype=torch.float64, device=x.device)
            codes[s["slots"].long()] = x / scale.unsqueeze(-1)
        got += [codes, pool]
    return got


def _rows64(s, n, b, length):
    """K or V of sequence b's first `length` cached tokens in 64 bits."""
    pt = s["pt"]
    pages = s["table"][b, :-(-length // pt)].long()
    slot = (pages.unsqueeze(1) * pt + torch.arange(pt, device=pages.device)).flatten()[:length]
    c = s[n + "_codes"]
    if s["kv"] == "f16":
        return c[slot].double()
    return c.view(torch.uint8)[slot].view(c.dtype).double() * s[n + "_scales"][slot].double().unsqueeze(-1)


def _exact_kv_gather(s, case):
    lens = _lengths(case)
    return [torch.cat([_rows64(s, n, b, length) for b, length in enumerate(lens)]) for n in "kv"]


def _exact_tree(s, case):
    bits = s["mask"].cpu().numpy().view(np.uint32)
    group, row, got = s["hq"] // s["hkv"], 0, []
    for b, (c, n) in enumerate(zip(_lengths(case), _drafted(case))):
        if n == 0:
            continue
        k, v = (_rows64(s, x, b, c + n).repeat_interleave(group, dim=1) for x in "kv")
        hide = torch.zeros((n, c + n), dtype=torch.bool)
        for j in range(n):
            hide[:, c + j] = torch.from_numpy((bits[row:row + n, j // 32] >> np.uint32(j % 32)) & 1 == 0)
        hide = hide.to(k.device).unsqueeze(0)
        score = torch.einsum("thd,shd->hts", s["qs"][row:row + n].double(), k) * s["scale"]
        p = torch.softmax(score.masked_fill(hide, -math.inf), dim=-1)
        p = p.masked_fill(hide.all(-1, keepdim=True), 0.0)
        got.append(torch.einsum("hts,shd->thd", p, v))
        row += n
    return torch.cat(got)


def _exact_logprobs(s):
    lp, order = [], []
    for x, mask in zip(s["logits"], s["mask"] if s["mask"] is not None else [None] * s["rows"]):
        x = x.double() * s["inv_t"]
        if mask is not None:
            words = torch.from_numpy(mask.cpu().numpy().view(np.uint8))
            ok = torch.from_numpy(np.unpackbits(words.numpy(), bitorder="little")[:s["vocab"]]).bool()
            x = x.masked_fill(~ok.to(x.device), -math.inf)
        y = torch.log_softmax(x, 0)
        p = y.exp()
        order.append(torch.cat([torch.special.xlogy(p, p).sum().neg().view(1), y.topk(s["top"]).values]))
        lp.append(y[s["tokens"][len(lp)].long()])
    order = torch.stack(order)
    return [torch.stack(lp), order[:, 0], order[:, 1:], None]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return _exact_rope(s)
    if op == "kv_append":
        return _exact_kv_append(s)
    if op == "kv_gather":
        return _exact_kv_gather(s, case)
    if op == "tree":
        return _exact_tree(s, case)
    return _exact_logprobs(s)
