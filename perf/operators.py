"""The operators of the 8-bit paged KV cache, as cases to be timed and compared.

The cache of one layer: e4m3 codes ``[pages, kv heads, page size, head_dim]`` for K and for
V, and one fp32 scale for each block (the tokens of one page, one kv head). A value is code
times scale; the scale is the smallest power of two that brings the block's largest
magnitude to 448 or less (0 for a block of zeros). Sequences list their pages in a CSR
(``kv_indptr``, ``kv_indices``, ``kv_last_page_len``); with ``qo_indptr`` the last ``qo_len``
positions of a sequence are new.

* ``append``: RoPE on q and k, then k and v quantised into the pages as they are written (an
  older token of a page is rounded again where a new one makes the block's scale grow),
  followed by reading back the pages that were written;
* ``gather``: pages read back as 16-bit values;
* ``decode``: attention of one query a sequence over its pages;
* ``prefill``: causal attention of a sequence's new rows over its pages.

With ``own`` the framework's entry points (``nanoslg_b200.ops``) are called, otherwise the
operators run as elementary torch operations in 32 bits.
"""
import math
import random

import torch

own = False

PAGE = 16
E4M3 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HEADS = [(32, 8), (16, 4), (8, 2), (4, 1), (16, 2), (64, 8), (8, 8)]


# ------------------------------------------------------------------------------ the cases
def listed():
    def c(name, kind, batch, lo, hi, new, hq=32, hkv=8, d=128, dtype="bf16"):
        return {"name": name, "kind": kind, "batch": batch, "len_min": lo, "len_max": hi, "new": new,
                "hq": hq, "hkv": hkv, "d": d, "dtype": dtype}
    return [
        # one user's token of an 8B-sized model, 513 tokens in: the latency of a step
        c("decode_1x513", "decode", 1, 513, 513, 1),
        # a step of 64 users of the 8B-sized model, 512-token prompts and up to 256 answered
        c("decode_64x768", "decode", 64, 513, 768, 1),
        # a long-context batch of the same layer, 512 to 8192 tokens a sequence (the largest)
        c("decode_64x8192", "decode", 64, 512, 8192, 1),
        # a shard of a 70B-sized model at four ranks (16 query, 2 kv heads), fp16, all lengths
        c("decode_32x4096_fp16", "decode", 32, 1, 4096, 1, hq=16, hkv=2, dtype="fp16"),
        # the new token of each of 64 sequences, at every place of a page
        c("append_64x1", "append", 64, 513, 768, 1),
        # the suffixes of 16 requests behind a shared prefix, fp16, starting inside a page
        c("append_16x128_fp16", "append", 16, 1150, 1165, 128, dtype="fp16"),
        # the prompts of a whole batch: 64 x 512 tokens
        c("append_64x512", "append", 64, 512, 512, 512),
        # a short sequence read back (a small model with head_dim 64)
        c("gather_1x300_d64", "gather", 1, 300, 300, 1, hq=4, hkv=2, d=64, dtype="fp16"),
        # 16 sequences with shared-prefix lengths read back
        c("gather_16x1152", "gather", 16, 1025, 1279, 1),
        # five rows checked at once against a long context (a guess of five tokens)
        c("prefill_1x5_of_4001_fp16", "prefill", 1, 4001, 4001, 5, dtype="fp16"),
        # suffixes of 128 tokens behind a cached prefix of 1024
        c("prefill_16x128_of_1152", "prefill", 16, 1152, 1152, 128),
        # the prompts of a whole batch: 64 x 512 tokens
        c("prefill_64x512", "prefill", 64, 512, 512, 512),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "append", "gather", "prefill", "prefill"])
    hq, hkv = rng.choice(HEADS)
    d = rng.choice([128, 128, 128, 64])
    dtype = rng.choice(["bf16", "fp16"])
    batch = _log(rng, 1, 64)
    if kind == "decode":
        hi = _log(rng, 1, 8192)
        new = 1
    elif kind == "gather":
        hi = _log(rng, 1, 2048)
        new = 1
    else:
        new = _log(rng, 1, 512)
        hi = new + (_log(rng, 1, 4096) if rng.random() < 0.6 else 0)
        # no more rows and no more scores than 64 prompts of 512 tokens have
        batch = max(1, min(batch, 32768 // new, (64 * 512 * 512 * 32) // (new * hi * hq)))
    batch = max(1, min(batch, (64 * 4352 * 8) // (hi * hkv)))
    lo = rng.randint(max(new, hi // 3), hi)
    return {"kind": kind, "batch": batch, "len_min": lo, "len_max": hi, "new": new, "hq": hq,
            "hkv": hkv, "d": d, "dtype": dtype}


def _lens(case):
    """Tokens of each sequence after the pass, a function of the case alone."""
    r = random.Random("%d %d %d" % (case["batch"], case["len_min"], case["len_max"]))
    return [r.randint(case["len_min"], case["len_max"]) for _ in range(case["batch"])]


def work(case):
    lens, new = _lens(case), case["new"]
    hq, hkv, d, es = case["hq"], case["hkv"], case["d"], 2
    toks = sum(lens)
    blocks = sum(-(-n // PAGE) for n in lens)
    plan = 4 * (blocks + 3 * len(lens))
    cache = 2 * hkv * (toks * d + 4 * blocks)               # codes and scales, read once
    if case["kind"] == "decode":
        return {"bytes": cache + plan + 2 * len(lens) * hq * d * es, "flops": 4 * hq * d * toks}
    if case["kind"] == "gather":
        return {"bytes": cache + plan + 2 * hkv * blocks * PAGE * d * es, "flops": 2 * hkv * toks * d}
    rows = new * len(lens)
    if case["kind"] == "prefill":
        seen = sum(new * (n - new) + new * (new + 1) // 2 for n in lens)
        return {"bytes": cache + plan + 2 * rows * hq * d * es, "flops": 4 * hq * d * seen}
    touched = sum(-(-n // PAGE) - (n - new) // PAGE for n in lens)
    written = 2 * hkv * (rows * d + 4 * touched)
    back = 2 * hkv * touched * PAGE * d * es
    tables = 2 * 4 * d * len({p for n in lens for p in range(n - new, n)})
    return {"bytes": rows * (2 * hq + 2 * hkv) * d * es + tables + written + 2 * hkv * touched * PAGE * d + back,
            "flops": 3 * rows * (hq + hkv) * d + 2 * rows * hkv * d}


# ------------------------------------------------------------------------------ the inputs
def _power(amax):
    """The smallest power of two s with amax <= 448 s; 0 for 0."""
    m, e = torch.frexp(amax)                                # amax = m 2^e, m in [1/2, 1)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e - 9 + (m > 0.875).to(e.dtype)),
                       torch.zeros_like(amax))


def _codes(x, scale):
    """x / scale as e4m3 (scale 0: a block of zeros)."""
    return (x / torch.where(scale > 0, scale, torch.ones_like(scale))).to(E4M3)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + 17)
    dt = TYPES[case["dtype"]]
    hq, hkv, d, new = case["hq"], case["hkv"], case["d"], case["new"]
    lens = _lens(case)
    n = torch.tensor(lens, device=dev)
    npg = (n + PAGE - 1) // PAGE
    total = int(npg.sum())
    pages = total + total // 4 + 2
    i32 = dict(dtype=torch.int32, device=dev)

    def csr(counts):
        out = torch.zeros(len(lens) + 1, **i32)
        out[1:] = counts.cumsum(0)
        return out

    # keys have channels that stand out, values do not; each kv head has a size of its own
    size = torch.exp2(torch.randn(hkv, 1, 1, device=dev, generator=g))
    channel = torch.exp(0.7 * torch.randn(hkv, 1, d, device=dev, generator=g)) * size
    s = {"case": dict(case), "hq": hq, "hkv": hkv, "d": d, "dtype": dt, "new": new, "max_len": max(lens),
         "sm_scale": 1.0 / math.sqrt(d), "batch": len(lens),
         "kv_indptr": csr(npg), "kv_last_page_len": (n - (npg - 1) * PAGE).to(torch.int32),
         "kv_indices": (torch.randperm(pages - 1, device=dev, generator=g)[:total] + 1).to(torch.int32),
         "qo_indptr": csr(torch.full_like(n, new))}
    for name, by in (("k", channel), ("v", size)):
        x = torch.randn(pages, hkv, PAGE, d, device=dev, generator=g) * by
        s["scale_" + name] = _power(x.abs().amax((2, 3)))
        s["pool_" + name] = _codes(x, s["scale_" + name][:, :, None, None])
        del x
    rows = new * len(lens)
    if case["kind"] != "gather":
        s["q"] = torch.randn(rows, hq, d, device=dev, generator=g).to(dt)
    if case["kind"] == "append":
        # the rows as a stacked q|k|v product leaves them: k and v are strided views
        kv = torch.randn(rows, 2 * hkv, d, device=dev, generator=g)
        kv[:, :hkv] *= channel[:, 0]
        kv[:, hkv:] *= size[:, 0]
        qkv = torch.cat([s["q"], kv.to(dt)], 1)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        ang = torch.outer(torch.arange(max(lens), device=dev, dtype=torch.float64),
                          500000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d))
        ang = torch.cat([ang, ang], 1)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        # the pages written by this pass, listed like the others, to be read back
        first = (n - new) // PAGE
        s["back_indptr"] = csr(npg - first)
        j = torch.arange(total, device=dev)
        b = torch.searchsorted(s["kv_indptr"][1:].contiguous(), j, right=True)
        s["back_indices"] = s["kv_indices"][j - s["kv_indptr"][b] >= first[b]].contiguous()
    return s


# ------------------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        from nanoslg_b200 import ops
        pool = (s["pool_k"], s["pool_v"], s["scale_k"], s["scale_v"])
        seqs = (s["kv_indptr"], s["kv_indices"], s["kv_last_page_len"])
        if kind == "decode":
            return ops.paged_decode_kv8(s["q"], *pool, *seqs, s["sm_scale"])
        if kind == "prefill":
            return ops.paged_prefill_kv8(s["q"], s["qo_indptr"], s["new"], *pool, *seqs, s["sm_scale"])
        if kind == "gather":
            return ops.kv8_gather(*pool, *seqs, s["dtype"])
        q = ops.rope_kv8_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], *pool, s["qo_indptr"], s["new"], *seqs)
        k, v = ops.kv8_gather(*pool, s["back_indptr"], s["back_indices"], s["kv_last_page_len"], s["dtype"])
        return q, k, v
    if kind == "decode" or kind == "prefill":
        return _attention(s)
    if kind == "gather":
        return _read(s, s["kv_indptr"], s["kv_indices"])
    q = _append(s)
    return (q, *_read(s, s["back_indptr"], s["back_indices"]))


def _pages(s, name, idx):
    """fp32 values [len(idx), hkv, PAGE, d] of the pages idx."""
    idx = idx.long()
    return s["pool_" + name].view(torch.uint8)[idx].view(E4M3).float() * s["scale_" + name][idx][:, :, None, None]


def _read(s, indptr, indices):
    j = torch.arange(indices.numel(), device=indices.device)
    b = torch.searchsorted(indptr[1:].contiguous(), j, right=True)
    fill = torch.where(j == indptr[b + 1] - 1, s["kv_last_page_len"][b], PAGE)
    held = (torch.arange(PAGE, device=indices.device) < fill[:, None])[:, :, None, None]
    return tuple(torch.where(held, _pages(s, name, indices).transpose(1, 2), 0.0).to(s["dtype"]).contiguous()
                 for name in ("k", "v"))


def _attention(s):
    """Rows padded to the longest sequence: [batch, hkv, rows x group, longest] scores."""
    B, hq, hkv, d, new = s["batch"], s["hq"], s["hkv"], s["d"], s["new"]
    npg = s["kv_indptr"][1:] - s["kv_indptr"][:-1]
    most = -(-s["max_len"] // PAGE)
    j = torch.arange(most, device=npg.device)
    idx = torch.where(j < npg[:, None], s["kv_indices"][(s["kv_indptr"][:-1, None] + j).clamp(max=s["kv_indices"].numel() - 1)], 0)
    length = (npg - 1) * PAGE + s["kv_last_page_len"]
    q = s["q"].float().view(B, new, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(B, hkv, -1, d)
    k = _pages(s, "k", idx.reshape(-1)).view(B, most, hkv, PAGE, d).transpose(1, 2).reshape(B, hkv, most * PAGE, d)
    p = torch.matmul(q, k.transpose(2, 3)) * s["sm_scale"]
    del k
    at = length[:, None] - new + torch.arange(new, device=npg.device)                    # [B, new]
    seen = torch.arange(most * PAGE, device=npg.device) <= at[:, :, None]                # [B, new, L]
    seen = seen[:, None, :, None].expand(B, 1, new, hq // hkv, most * PAGE).reshape(B, 1, -1, most * PAGE)
    p = p.masked_fill_(~seen, float("-inf"))
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = _pages(s, "v", idx.reshape(-1)).view(B, most, hkv, PAGE, d).transpose(1, 2).reshape(B, hkv, most * PAGE, d)
    o = torch.matmul(p, v)
    return o.view(B, hkv, new, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(B * new, hq, d).to(s["dtype"])


def _append(s):
    B, new, hkv = s["batch"], s["new"], s["hkv"]
    dev = s["q"].device
    npg = s["kv_indptr"][1:] - s["kv_indptr"][:-1]
    length = (npg - 1) * PAGE + s["kv_last_page_len"]
    pos = (length[:, None] - new + torch.arange(new, device=dev)).reshape(-1)            # of each row
    b = torch.arange(B, device=dev).repeat_interleave(new)
    page = s["kv_indices"][s["kv_indptr"][b] + pos // PAGE].long()
    slot = pos % PAGE
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def rotated(x):
        x = x.float()
        x1, x2 = x.chunk(2, -1)
        return x * cos + torch.cat([-x2, x1], -1) * sin

    start = (length - new)[b]
    older = (pos // PAGE == start // PAGE) & (start % PAGE > 0)       # the page has tokens before this pass
    for name, x in (("k", rotated(s["k"])), ("v", s["v"].float())):
        pool, scale = s["pool_" + name], s["scale_" + name]
        fresh = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(-1), "amax")
        kept = torch.zeros_like(scale).index_reduce_(0, page, scale[page] * older[:, None], "amax")
        grown = torch.maximum(_power(fresh), kept)
        touched = s["back_indices"].long()
        codes = _codes(_pages(s, name, touched), grown[touched][:, :, None, None])
        pool.view(torch.uint8)[touched] = codes.view(torch.uint8)
        scale[touched] = grown[touched]
        codes = _codes(x, grown[page][:, :, None])
        pool.view(torch.uint8)[page[:, None], torch.arange(hkv, device=dev), slot[:, None]] = codes.view(torch.uint8)
    return rotated(s["q"]).to(s["dtype"])


# ------------------------------------------------------------------------------ in 64 bits
def _exact_e4m3(y):
    """y rounded to the nearest e4m3 value, ties to the even one, |y| <= 448."""
    e = torch.frexp(y)[1] - 1
    step = torch.ldexp(torch.ones_like(y), e.clamp(min=-6) - 3)
    return torch.round(y / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    kind, lens, new = case["kind"], _lens(case), case["new"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    ptr = [0]
    for n in lens:
        ptr.append(ptr[-1] + -(-n // PAGE))
    indices = s["kv_indices"].long()

    def held(name, b, first=0):
        """Sequence b's tokens from page ``first`` of its list on: [tokens, hkv, d], 64 bits."""
        idx = indices[ptr[b] + first:ptr[b + 1]]
        x = s["pool_" + name].view(torch.uint8)[idx].view(E4M3).double() * s["scale_" + name][idx].double()[:, :, None, None]
        return x.permute(0, 2, 1, 3).reshape(-1, hkv, d)[:lens[b] - first * PAGE]

    def paged(x):
        """[tokens, hkv, d] as whole pages, zeros behind the last token."""
        full = torch.zeros(-(-x.shape[0] // PAGE) * PAGE, hkv, d, dtype=torch.float64, device=x.device)
        full[:x.shape[0]] = x
        return full.view(-1, PAGE, hkv, d)

    if kind == "gather":
        return tuple(torch.cat([paged(held(name, b)) for b in range(len(lens))]) for name in ("k", "v"))
    if kind in ("decode", "prefill"):
        out = torch.empty(len(lens) * new, hq, d, dtype=torch.float64, device="cuda")
        for b, n in enumerate(lens):
            k, v = held("k", b), held("v", b)
            seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - new, n, device="cuda")[:, None]
            for h in range(hq):
                q = s["q"][b * new:(b + 1) * new, h].double()
                w = (q @ k[:, h * hkv // hq].T) * s["sm_scale"]
                out[b * new:(b + 1) * new, h] = torch.softmax(w.masked_fill(~seen, -math.inf), -1) @ v[:, h * hkv // hq]
        return out
    half = d // 2
    cos, sin = s["cos"].double(), s["sin"].double()

    def turn(x, lo):
        c, r = cos[lo:lo + new, None], sin[lo:lo + new, None]
        x = x.double()
        return torch.cat([x[..., :half] * c[..., :half] - x[..., half:] * r[..., :half],
                          x[..., half:] * c[..., half:] + x[..., :half] * r[..., half:]], -1)

    qs, ks, vs = [], [], []
    for b, n in enumerate(lens):
        rows, lo = slice(b * new, (b + 1) * new), n - new
        qs.append(turn(s["q"][rows], lo))
        first = lo // PAGE
        for name, x, back in (("k", turn(s["k"][rows], lo), ks), ("v", s["v"][rows].double(), vs)):
            old = held(name, b, first)[:lo - first * PAGE]
            was = s["scale_" + name][indices[ptr[b] + first]].double() if lo % PAGE else torch.zeros(hkv, device="cuda", dtype=torch.float64)
            fresh = torch.cat([torch.zeros_like(old), x])
            every = paged(torch.cat([old, x]))
            amax = paged(fresh).abs().amax((1, 3))                                       # [pages, hkv]
            by = torch.where(amax > 0, torch.exp2(torch.ceil(torch.log2(amax / 448))), 0.0)
            by = torch.where(by * 224 >= amax, by / 2, by)                               # log2 was a step too high
            by = torch.where(by * 448 < amax, by * 2, by)                                # ... or too low
            by[0] = torch.maximum(by[0], was)
            by = by[:, None, :, None]
            safe = torch.where(by > 0, by, 1.0)
            back.append(_exact_e4m3(every / safe) * by)
    return torch.cat(qs), torch.cat(ks), torch.cat(vs)
