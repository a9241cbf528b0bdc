"""The 8-bit cache without a GPU: the oracle's rounding and scales, and what the entry
points refuse."""
import ctypes
import math
import os
import re
import sysconfig
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from nanoslg_b200 import _native as N
from nanoslg_b200 import build, ops
from oracle import kv8


@pytest.fixture(scope="module")
def lib():
    build.build()
    return N.lib()


def test_oracle_rounding_is_e4m3():
    every = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    finite = np.sort(every[np.isfinite(every)])
    np.testing.assert_array_equal(kv8.e4m3(finite), finite)
    # neighbours' middles: a tie goes to the even code, anything off it to the nearer one
    lo, hi = finite[:-1], finite[1:]
    mid = (lo + hi) / 2
    want = torch.from_numpy(mid).to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(kv8.e4m3(mid), want)
    np.testing.assert_array_equal(np.abs(kv8.e4m3(np.nextafter(mid, hi)) - hi).max(), 0)
    np.testing.assert_array_equal(np.abs(kv8.e4m3(np.nextafter(mid, lo)) - lo).max(), 0)


@pytest.mark.parametrize("amax,scale", [(0.0, 0.0), (448.0, 1.0), (448.0001, 2.0), (224.0, 0.5),
                                        (1.0, 2.0 ** -8), (1.75, 2.0 ** -8), (1.7501, 2.0 ** -7),
                                        (3.4e38, 2.0 ** 120), (1e-45, 2.0 ** -126),
                                        (math.inf, math.nan), (math.nan, math.nan)])
def test_oracle_scale(amax, scale):
    got = kv8.scale_of(amax)
    assert (math.isnan(got) and math.isnan(scale)) or got == scale


def test_oracle_append_does_not_depend_on_the_cut_but_for_subnormals():
    rng = np.random.default_rng(0)
    k = rng.standard_normal((40, 2, 32)) * np.exp2(rng.integers(-1, 2, (40, 2, 1)))
    whole, single = (kv8.Cache(4, 2, 16, 32) for _ in range(2))
    whole.append([3, 1, 2], 0, k, k)
    for t in range(40):
        single.append([3, 1, 2], t, k[t:t + 1], k[t:t + 1])
    np.testing.assert_array_equal(whole.s["k"], single.s["k"])
    a, b = whole.read([3, 1, 2], 40, "k"), single.read([3, 1, 2], 40, "k")
    s = np.repeat(whole.s["k"][[3, 1, 2]], 16, 0)[:40, :, None]
    normal = np.abs(k) >= s * 2.0 ** -6
    np.testing.assert_array_equal(a[normal], b[normal])
    assert (np.abs(a - b) <= s * 2.0 ** -9)[~normal].all()


def _attend(lib, dtype=N.DTYPE_BF16, batch=1, hq=8, hkv=2, d=128, ps=16, q=16, qs=1024, out=16,
            pool=16, scale=16, pages=4, plan=16, sm=0.1, name="nslg_paged_decode_kv8"):
    vp = ctypes.c_void_p
    return lib.nslg_paged_decode_kv8(dtype, batch, hq, hkv, d, ps, vp(q), qs, vp(out), qs, vp(pool),
                                     vp(pool), vp(scale), vp(scale), pages, vp(plan), vp(plan),
                                     vp(plan), sm, None, 0, None, None)


@pytest.mark.parametrize("bad,what", [
    (dict(dtype=7), b"dtype"), (dict(batch=-1), b"batch"), (dict(hkv=0), b"num_kv_heads"),
    (dict(hq=9), b"num_qo_heads"), (dict(d=40), b"head_dim"), (dict(d=288), b"head_dim"),
    (dict(ps=0), b"page_size"), (dict(pages=0), b"num_pages"), (dict(pool=0), b"null cache"),
    (dict(scale=0), b"null cache"), (dict(plan=0), b"page list"), (dict(pool=24), b"aligned"),
    (dict(q=0), b"null"), (dict(out=0), b"null"), (dict(q=18), b"aligned"), (dict(qs=1020), b"stride"),
    (dict(qs=512), b"stride"), (dict(sm=0.0), b"sm_scale"), (dict(sm=math.nan), b"sm_scale"),
    (dict(ps=65536, hq=256, hkv=256, qs=32768), b"2^31 elements"), (dict(ps=65537), b"page_size")])
def test_attention_refusals(lib, bad, what):
    assert _attend(lib, **bad) in (N.ERR_ARG, N.ERR_UNSUPPORTED)
    assert what in lib.nslg_last_error()


def test_empty_calls_do_nothing(lib):
    assert _attend(lib, batch=0, q=0, out=0, pool=0) == N.OK
    z = [None] * 2
    assert lib.nslg_kv8_gather(N.DTYPE_F32, 0, 2, 64, 16, *z, *z, 4, *z, None, 8, *z, None, None) == N.OK
    assert lib.nslg_rope_kv8_append(N.DTYPE_F32, 1, 2, 2, 64, 16, None, 0, None, 0, None, 0, 0, None,
                                    None, None, 0, None, None, None, None, 4, None, None, 0, None,
                                    None, None, None, None) == N.OK


@pytest.mark.parametrize("bad,what", [
    (dict(cos=0), b"cos and sin"), (dict(rows=0), b"cos and sin"), (dict(k=0), b"null"),
    (dict(q=0), b"q_out given without q"), (dict(qo=0), b"null"), (dict(most=-1), b"max_qo_len"),
    (dict(ks=100), b"k rows"), (dict(v=8), b"v rows"), (dict(cos=20), b"tables")])
def test_append_refusals(lib, bad, what):
    a = dict(q=16, k=16, v=16, ks=256, cos=16, rows=5, qo=16, most=4) | bad
    vp = ctypes.c_void_p
    rc = lib.nslg_rope_kv8_append(N.DTYPE_BF16, 1, 8, 2, 128, 16, vp(a["q"]), 1024, vp(a["k"]), a["ks"],
                                  vp(a["v"]), 256, 4, vp(16), vp(a["cos"]), vp(16), a["rows"], vp(16),
                                  vp(16), vp(16), vp(16), 4, vp(a["qo"]), None, a["most"], vp(16),
                                  vp(16), vp(16), None, None)
    assert rc == N.ERR_ARG and what in lib.nslg_last_error()


def test_gather_and_prefill_refusals(lib):
    vp = ctypes.c_void_p
    p = vp(16)
    rc = lib.nslg_kv8_gather(N.DTYPE_BF16, 1, 2, 128, 16, p, p, p, p, 4, p, p, p, 8, None, p, None, None)
    assert rc == N.ERR_ARG and b"null" in lib.nslg_last_error()
    rc = lib.nslg_kv8_gather(N.DTYPE_BF16, 1, 2, 128, 16, p, p, p, p, 4, p, p, p, -1, p, p, None, None)
    assert rc == N.ERR_ARG and b"num_indices" in lib.nslg_last_error()
    rc = lib.nslg_paged_prefill_kv8(N.DTYPE_BF16, 1, 8, 2, 128, 16, p, 1024, 0, p, 1024, p, None, 4, p,
                                    p, p, p, 4, p, p, p, 0.1, 1, None, 0, None, None)
    assert rc == N.ERR_ARG and b"q_rows" in lib.nslg_last_error()
    rc = lib.nslg_paged_prefill_kv8(N.DTYPE_BF16, 1, 8, 2, 128, 16, p, 1024, 4, p, 1024, None, None, 4,
                                    p, p, p, p, 4, p, p, p, 0.1, 1, None, 0, None, None)
    assert rc == N.ERR_ARG and b"null" in lib.nslg_last_error()


def _calls(row, pool, i, bad):
    """The four operators on one row, with arguments replaced by name."""
    a = dict(q=row, k=row[:, :2], v=row[:, :2], cos=torch.zeros(8, 64), sin=torch.zeros(8, 64), pool_k=pool[0],
             pool_v=pool[1], scale_k=pool[2], scale_v=pool[3], qo_indptr=i, max_qo_len=1, kv_indptr=i,
             kv_indices=i, kv_last_page_len=i, sm_scale=0.1, dtype=torch.bfloat16, out=None, q_out=None) | bad
    cache = [a[n] for n in ("pool_k", "pool_v", "scale_k", "scale_v")]
    seqs = [a[n] for n in ("kv_indptr", "kv_indices", "kv_last_page_len")]
    return {"append": lambda: ops.rope_kv8_append(a["q"], a["k"], a["v"], a["cos"], a["sin"], *cache,
                                                  a["qo_indptr"], a["max_qo_len"], *seqs, q_out=a["q_out"],
                                                  q_row_start=a.get("q_row_start")),
            "gather": lambda: ops.kv8_gather(*cache, *seqs, a["dtype"], out=a["out"]),
            "decode": lambda: ops.paged_decode_kv8(a["q"], *cache, *seqs, a["sm_scale"], out=a["out"]),
            "prefill": lambda: ops.paged_prefill_kv8(a["q"], a["qo_indptr"], a["max_qo_len"], *cache, *seqs,
                                                     a["sm_scale"], out=a["out"],
                                                     q_row_start=a.get("q_row_start"))}


EVERY = ("append", "gather", "decode", "prefill")
POOL = ops.kv8_pages(4, 16, 2, 64, "cpu")
Q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
I = torch.zeros(2, dtype=torch.int32)


@pytest.mark.parametrize("names,bad,error,what", [
    (EVERY, dict(), RuntimeError, "CUDA"),
    (EVERY, dict(pool_k=POOL[0].float()), TypeError, "float8_e4m3fn"),
    (EVERY, dict(pool_v=POOL[1].view(torch.uint8)), TypeError, "float8_e4m3fn"),
    (EVERY, dict(pool_v=POOL[1][:3]), ValueError, "alike"),
    (EVERY, dict(pool_k=POOL[0][0]), ValueError, "alike"),
    (EVERY, dict(pool_k=POOL[0].transpose(2, 3), pool_v=POOL[1].transpose(2, 3)), ValueError, "contiguous"),
    (EVERY, dict(scale_k=POOL[2].double()), ValueError, "scales"),
    (EVERY, dict(scale_v=POOL[3][:, :1]), ValueError, "scales"),
    (EVERY, dict(scale_v=POOL[3].t().contiguous().t()), ValueError, "scales"),
    (EVERY, dict(kv_indices=I.long()), ValueError, "int32"),
    (EVERY, dict(kv_indptr=torch.zeros(4, dtype=torch.int32)), ValueError, "entries"),
    (EVERY, dict(kv_indptr=torch.zeros(0, dtype=torch.int32)), ValueError, "entries"),
    (EVERY, dict(pool_k=None), TypeError, "pool_k"),
    (("append", "decode", "prefill"), dict(q=torch.zeros(1, 3, 64, dtype=torch.bfloat16)), ValueError, "kv heads"),
    (("append", "decode", "prefill"), dict(q=torch.zeros(1, 4, 32, dtype=torch.bfloat16)), ValueError, "kv heads"),
    (("append", "decode", "prefill"), dict(q=torch.zeros(4, 64, dtype=torch.bfloat16)), ValueError, "kv heads"),
    (("append", "decode", "prefill"), dict(q=torch.zeros(1, 64, 4, dtype=torch.bfloat16).transpose(1, 2)),
     ValueError, "contiguous"),
    (("append", "decode", "prefill"), dict(q=torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16).expand(3, 2, 4, 64)),
     ValueError, "."),
    (("decode", "prefill"), dict(q=Q.double()), TypeError, "bfloat16, float16 and float32"),
    (("gather",), dict(dtype=torch.float64), TypeError, "bfloat16, float16 and float32"),
    (("gather",), dict(dtype="bf16"), TypeError, "dtype"),
    (("gather",), dict(out=(Q, Q)), ValueError, "outputs"),
    (("decode",), dict(q=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), ValueError, "2 queries for 1"),
    (("decode", "prefill"), dict(out=Q.float()), ValueError, "out must"),
    (("decode", "prefill"), dict(out=torch.zeros(2, 4, 64, dtype=torch.bfloat16)), ValueError, "out must"),
    (("decode", "prefill"), dict(sm_scale="x"), TypeError, "."),
    (("append", "prefill"), dict(qo_indptr=torch.zeros(3, dtype=torch.int32)), ValueError, "qo_indptr"),
    (("append", "prefill"), dict(q_row_start=I), ValueError, "q_row_start"),
    (("append", "prefill"), dict(max_qo_len=1 << 40), ValueError, "range"),
    (("append",), dict(k=Q), ValueError, "kv heads"),
    (("append",), dict(v=Q[:, :2].float()), ValueError, "same rows"),
    (("append",), dict(q=Q.float()), ValueError, "q must match"),
    (("append",), dict(q=None, q_out=Q), ValueError, "without q"),
    (("append",), dict(q_out=Q.float()), ValueError, "q_out must"),
    (("append",), dict(cos=None), ValueError, "cos/sin"),
    (("append",), dict(sin=torch.zeros(8, 32)), ValueError, "cos/sin"),
    (("append",), dict(cos=torch.zeros(8, 64).double()), ValueError, "cos/sin"),
])
def test_ops_refuse(lib, names, bad, error, what):
    """Layouts and types are refused before the device is looked at; sound CPU tensors then are
    for being on the CPU."""
    calls = _calls(Q, POOL, I, bad)
    for n in names:
        with pytest.raises(error, match=what):
            calls[n]()


def _split(total, n):
    """Bounds of n contiguous parts of [0, total), the first total % n one longer."""
    q, r = divmod(total, n)
    return [q * c + min(c, r) for c in range(n + 1)]


def _leaves_early():
    """The condition under which a CTA of the split kernel ends before it arrives, from the source."""
    path = os.path.join(os.path.dirname(N.__file__), "csrc", "kv8_attn_tc.cu")
    with open(path) as f:
        body = f.read().split("const int ngroups = s_ngroups;")[1].split("atom_add_acq_rel_u32")[0]
    found = re.findall(r"if \((.*)\) return;", body)
    assert len(found) == 1
    text = found[0].replace("&&", "and").replace("s_join[0].vid", "vid0").replace("s_join[1].vid", "vid1")
    return compile(text, path, "eval")


@pytest.mark.parametrize("seed", range(40))
def test_split_attention_counts_return_to_zero_when_warps_give_up(seed):
    """A model of the split kernel's bookkeeping: every CTA over which a virtual sequence is spread
    arrives at the count of its first one, wherever the waits of any warps ran out (a warp that
    gives up leaves a piece of the sequence it was at and none of those behind it)."""
    rng = np.random.default_rng(seed)
    leaves = _leaves_early()
    hm, warps, sms = int(rng.integers(1, 9)), 12, int(rng.integers(2, 20))
    pages = rng.integers(0, 40, int(rng.integers(1, 6)))
    if seed % 2:                                    # many sequences of a page before a long one
        pages = np.array([1] * int(rng.integers(20, 60)) + [400])
    starts = np.cumsum([0] + [n for n in pages for _ in range(hm)])       # first unit of each sequence
    total = int(starts[-1])
    vid_of = [v for v in range(len(starts) - 1) for _ in range(starts[v + 1] - starts[v])]
    n = min(-(-total // warps), sms)
    if n == 0:
        return
    ctas = _split(total, n)
    cta_of = [c for c in range(n) for _ in range(ctas[c + 1] - ctas[c])]
    arrived, expected = [0] * n, [0] * n
    for v in range(len(starts) - 1):
        if starts[v] < starts[v + 1]:
            first, last = cta_of[starts[v]], cta_of[starts[v + 1] - 1]
            expected[first] += last - first + 1 if last > first else 0
    for c in range(n):
        u0, u1 = ctas[c], ctas[c + 1]
        head, tail = vid_of[u0], vid_of[u1 - 1]
        joins = [head if starts[head] < u0 else -1,
                 tail if starts[tail] >= u0 and starts[tail + 1] > u1 else -1]
        groups = set()
        for a, b in zip(*(lambda w: (w, w[1:]))([u0 + x for x in _split(u1 - u0, warps)])):
            # units it got through
            stop = a if seed % 2 else int(rng.integers(a, b + 1)) if rng.random() < 0.7 else b
            for v in set(vid_of[a:min(stop + 1, b)]):
                if starts[v] < a or starts[v + 1] > b:                       # not whole: a piece
                    groups.add(v)
        if eval(leaves, {}, {"ngroups": len(groups), "vid0": joins[0], "vid1": joins[1]}):
            continue
        for v in joins:
            if v >= 0:
                arrived[cta_of[starts[v]]] += 1
    assert arrived == expected


def test_the_torch_side_is_built_again_for_another_torch_or_python(monkeypatch, tmp_path):
    """Version A, B and A again: three compilations, none while nothing changes."""
    runs = []

    def compile_(cmd, **_):
        runs.append(cmd)
        (tmp_path / "_kv8.so").write_text("built")
        return SimpleNamespace(returncode=0)
    monkeypatch.setattr(build, "KV8", str(tmp_path / "_kv8.so"))
    monkeypatch.setattr(build, "BUILD", str(tmp_path))
    monkeypatch.setattr(build.subprocess, "run", compile_)
    for version in ("2.0", "2.0", "2.1", "2.1", "2.0", "2.0"):
        monkeypatch.setattr(torch, "__version__", version)
        build.build_torch()
    assert len(runs) == 3
    monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "another python")
    build.build_torch()
    build.build_torch()
    assert len(runs) == 4


def test_manager_bookkeeping_does_not_depend_on_the_cache_type():
    """Pages, plans and copy on write of an 8-bit pool on the CPU: the ids of a 16-bit one, and
    a copied page takes its scales along."""
    from nanoslg_b200.kv_cache import B200PagedKVCache, KVCacheConfig
    mgrs = [B200PagedKVCache(KVCacheConfig(num_layers=2, num_kv_heads=2, num_qo_heads=4, head_dim=32,
                                           page_size=4, max_pages=40, dtype=torch.bfloat16, kv_dtype=t))
            for t in (None, "fp8")]
    assert mgrs[0].pool.kv8_layers is None
    assert mgrs[1].pool.k.shape == (2, 40, 2, 4, 32) and mgrs[1].pool.k.dtype == torch.float8_e4m3fn
    plans = []
    for m in mgrs:
        m.allocate_sequence("a", list(range(11)))
        m.begin_forward(["a"], [11])
        m.seqs["a"].num_tokens = 11
        m.release_sequence("a")
        n = m.allocate_sequence("b", list(range(11)))
        m.seqs["b"].num_tokens = n - 1
        page = m.seqs["b"].block_table[1]
        if m.pool.kv8_layers:
            m.pool.k_scale[:, page] = 3.0
            m.pool.v_scale[:, page] = 5.0
            m.pool.k.view(torch.uint8)[:, page] = 7
        ctx = m.begin_forward(["b"], [2])
        assert m.seqs["b"].block_table[1] != page
        plans.append((list(m.seqs["b"].block_table), ctx.kv_indptr.tolist(), ctx.kv_indices.tolist(),
                      ctx.kv_last_page_len.tolist(), ctx.qo_indptr.tolist(), ctx.q_row_start.tolist()))
    assert plans[0] == plans[1]
    new = mgrs[1].seqs["b"].block_table[1]
    assert bool((mgrs[1].pool.k_scale[:, new] == 3.0).all()) and bool((mgrs[1].pool.v_scale[:, new] == 5.0).all())
    assert bool((mgrs[1].pool.k.view(torch.uint8)[:, new] == 7).all())


@pytest.mark.parametrize("kv_dtype,ok", [(None, True), ("auto", True), ("fp8", True), ("fp8_e4m3", True),
                                         (torch.float8_e4m3fn, True), ("int8", False),
                                         (torch.float8_e5m2, False)])
def test_kv_dtype_names(kv_dtype, ok):
    from nanoslg_b200.kv_cache import KVCacheConfig

    def make(d=64):
        return KVCacheConfig(num_layers=1, num_kv_heads=1, num_qo_heads=1, head_dim=d, kv_dtype=kv_dtype)
    if not ok:
        with pytest.raises(ValueError, match="kv cache dtype"):
            make()
        return
    assert make().kv8 == (kv_dtype not in (None, "auto"))
    if make().kv8:
        with pytest.raises(ValueError, match="head_dim"):
            make(d=80)
