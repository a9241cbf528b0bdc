"""Seeded problems over the 8-bit KV cache and the tolerances of its tests."""
import numpy as np
import torch

from oracle import kv8

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def page_lists(lens, page_size, num_pages, seed):
    """Random distinct pages (never page 0) of sequences of these lengths."""
    rng = np.random.default_rng(seed)
    npg = [-(-n // page_size) for n in lens]
    ids = rng.permutation(num_pages - 1)[:sum(npg)] + 1
    ends = np.cumsum([0] + npg)
    return [ids[a:b].astype(np.int32) for a, b in zip(ends, ends[1:])]


def csr(tables, lens, page_size, device, spare=0):
    """kv_indptr, kv_indices (``spare`` entries behind the list, outside any pool), lpl."""
    ptr = np.cumsum([0] + [len(t) for t in tables]).astype(np.int32)
    idx = np.concatenate(list(tables) + [np.full(spare, 1 << 30, np.int32)]).astype(np.int32)
    lpl = np.array([n - (len(t) - 1) * page_size if len(t) else 0 for t, n in zip(tables, lens)],
                   dtype=np.int32)
    return tuple(torch.from_numpy(a).to(device) for a in (ptr, idx if idx.size else np.zeros(1, np.int32), lpl))


def rows(shape, dtype, seed, spread=0.0):
    """N(0, 1) rows of ``dtype``; with ``spread`` each head row has a magnitude of its own."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if spread:
        x = x * torch.exp2(spread * torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(dtype)


def idle_for_tiles(batch, hq, hkv, max_qo_len, sms=148):
    """How many sequences without rows and pages make a prefill of ``batch`` large enough for
    the kernel that works on tiles of 256 query rows (each kv head of a sequence counts as
    if it had max_qo_len rows); None where none do."""
    rows = max_qo_len * (hq // hkv)
    tiles, pairs = -(-rows // 16), -(-rows // 256)
    for idle in range(400):
        vs = (batch + idle) * hkv
        if vs * tiles > 2 * sms * -(-pairs * vs // sms):
            return idle
    return None


def random_cache(num_pages, hkv, page_size, d, device, seed, power=True):
    """A pool of random finite codes, its scales powers of two (any value unless ``power``)."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        codes = (torch.randn((num_pages, hkv, page_size, d), generator=g) * 120).clamp(-448, 448)
        out.append(codes.to(torch.float8_e4m3fn).to(device))
    for _ in range(2):
        s = torch.exp2(torch.randint(-8, -4, (num_pages, hkv), generator=g).float())
        if not power:
            s = s * (1 + torch.rand((num_pages, hkv), generator=g))
        out.append(s.to(device))
    return tuple(out)


def values(pool, scale, table, length):
    """[length, hkv, d] in 64 bits of the pages ``table`` of a pool."""
    idx = torch.from_numpy(np.asarray(table)).long()
    x = pool.view(torch.uint8).cpu()[idx].view(torch.float8_e4m3fn).double()
    x = x * scale.cpu()[idx].double()[:, :, None, None]
    return x.permute(0, 2, 1, 3).reshape(-1, pool.shape[1], pool.shape[3])[:length].numpy()


def attention_bound(q, k, v, vs, sm_scale, out, dtype, p_half, causal=True):
    """How far an output may be from the 64-bit ``out``, per element: the output rounded once
    (half a step of its type; 2^-25 where fp16 is subnormal), plus, relative to A = sum p |v|:
    the weights rounded to the type the products take (p_half), the fp32 score (D products of
    at most S in all, each sum rounded), the exponential's argument (2^-24 of up to log2(e) S
    and of the scales' exponents, its own 2^-22) and the fp32 sums over the keys (at most one
    rounding a key, numerator and denominator); plus, for weights p scale_v that are fp16
    subnormals beside the row's largest W, at most 2^-25 W times the key's code.
    ``vs`` [tokens, hkv]: the scales of the V blocks."""
    n, hq, d = q.shape
    length, hkv = k.shape[0], k.shape[1]
    a = kv8.attention(q, k, np.abs(v), sm_scale, causal)
    w = np.zeros_like(a)
    s = 0.0
    for h in range(hq):
        if not length:
            break
        kh = h * hkv // hq
        s = max(s, float((np.abs(q[:, h]) @ np.abs(k[:, kh]).T).max()) * sm_scale)
        # p scale_v: attention over the diagonal matrix of the scales
        one = kv8.attention(q[:, h:h + 1], k[:, kh:kh + 1], np.diag(vs[:, kh])[:, None], sm_scale, causal)
        codes = np.abs(v[:, kh]) / np.where(vs[:, kh] > 0, vs[:, kh], 1.0)[:, None]
        w[:, h] = one[:, 0].max(1, keepdims=True) * codes.sum(0)[None]
    rel = p_half + (d + 40) * s * 2.0 ** -24 + 2.0 ** -19 + 2 * length * 2.0 ** -24
    half = HALF[dtype] * np.abs(out) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    return half + rel * a + (2.0 ** -25 * w if p_half else 0.0) + 1e-30


def token_scales(scale, table, length, page_size):
    """[length, hkv] scales of a sequence's tokens in 64 bits."""
    return np.repeat(scale.cpu().double().numpy()[np.asarray(table, dtype=int)], page_size, 0)[:length]
