"""The 8-bit KV cache on the GPU against its 64-bit definition (oracle/kv8.py).

The append is compared bit for bit: scales, codes and q follow from fp32 operations whose
rounding is fixed. Attention tolerances are derived in kv8_util.attention_bound."""
import math

import numpy as np
import pytest
import torch

import kv8_util as U
from nanoslg_b200 import ops
from oracle import kv8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _clean_status():
    ops.status_word(DEV).zero_()
    yield
    ops.check_device_status(DEV)


def _tables(rows, d):
    ang = torch.outer(torch.arange(rows, dtype=torch.float64),
                      10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d))
    ang = torch.cat([ang, ang], 1)
    return ang.cos().float(), ang.sin().float()


def _append(cache, oracle, tables, starts, counts, hq, dt, seed, rope, ps, left=0, spread=1.0):
    """One append of counts[b] tokens behind starts[b], on the kernel and on the oracle; rows
    are left padded by ``left``. Returns (q_out, expected q_out) of the real rows."""
    hkv, d = cache[0].shape[1], cache[0].shape[3]
    lens = [s + n for s, n in zip(starts, counts)]
    width = max(counts) + left
    row_start = [b * width + width - n for b, n in enumerate(counts)]
    q = U.rows((len(lens) * width, hq, d), dt, seed, spread)
    k = U.rows((len(lens) * width, hkv, d), dt, seed + 1, spread)
    v = U.rows((len(lens) * width, hkv, d), dt, seed + 2, spread)
    cos, sin = _tables(max(lens) + 1, d)
    npg = [-(-n // ps) for n in lens]
    ptr, idx, lpl = U.csr([t[:n] for t, n in zip(tables, npg)], lens, ps, DEV, spare=3)
    qo = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=DEV)
    got = ops.rope_kv8_append(q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), *cache, qo,
                              max(counts), ptr, idx, lpl,
                              q_row_start=torch.tensor(row_start, dtype=torch.int32, device=DEV),
                              rotate=rope).cpu()
    mine, want = [], []
    for b, (s, n) in enumerate(zip(starts, counts)):
        r = slice(row_start[b], row_start[b] + n)
        kf, qf = k[r].float().numpy(), q[r].float().numpy()
        if rope:
            c, t = cos[s:s + n].numpy(), sin[s:s + n].numpy()
            kf, qf = kv8.rotate(kf, c, t), kv8.rotate(qf, c, t)
        oracle.append(tables[b], s, kf, v[r].float().numpy())
        mine.append(got[r])
        want.append(torch.from_numpy(qf).to(dt))
    return torch.cat(mine), torch.cat(want)


def _assert_cache(cache, oracle, tables, lens):
    for i, name in enumerate("kv"):
        for t, n in zip(tables, lens):
            t = t[:-(-n // oracle.ps)]
            np.testing.assert_array_equal(cache[2 + i].cpu().numpy()[t], oracle.s[name][t])
            np.testing.assert_array_equal(U.values(cache[i], cache[2 + i], t, n),
                                          oracle.read(t, n, name))


APPEND = [
    # dtype, hq, hkv, d, page size, starts, counts, rope
    (torch.bfloat16, 32, 8, 128, 16, [0, 0, 0], [1, 16, 33], True),
    (torch.bfloat16, 32, 8, 128, 16, [5, 15, 16, 100], [1, 1, 1, 1], True),
    (torch.float16, 8, 2, 64, 16, [3, 31, 0], [40, 1, 17], True),
    (torch.float16, 16, 2, 128, 16, [7, 8], [1, 1], True),
    (torch.bfloat16, 4, 4, 64, 16, [1, 2, 0], [1, 1, 1], True),
    (torch.float32, 4, 2, 64, 16, [0, 9], [25, 3], True),
    (torch.float32, 4, 2, 64, 16, [4, 9], [1, 1], True),
    (torch.bfloat16, 6, 3, 96, 5, [0, 4, 12], [11, 1, 2], True),
    (torch.float16, 5, 5, 32, 1, [0, 3], [4, 1], True),
    (torch.bfloat16, 64, 4, 128, 16, [12, 0], [70, 2], False),
    (torch.bfloat16, 2, 1, 256, 64, [60, 0], [9, 130], True),
]


@pytest.mark.parametrize("dt,hq,hkv,d,ps,starts,counts,rope", APPEND)
def test_append_is_the_definition(dt, hq, hkv, d, ps, starts, counts, rope):
    lens = [s + n for s, n in zip(starts, counts)]
    pages = sum(-(-n // ps) for n in lens) + 5
    tables = U.page_lists(lens, ps, pages, 1)
    cache = U.random_cache(pages, hkv, ps, d, DEV, 2)           # leftovers in every page
    cache[0].view(torch.uint8)[:, :, ps - 1] = 0x7F             # NaN codes among them
    oracle = kv8.Cache(pages, hkv, ps, d)
    before = [t.clone() for t in cache]
    if any(starts):
        first = [s if s else 1 for s in starts]                 # every page list gets a start
        _append(cache, oracle, tables, [0] * len(lens), [min(f, n) for f, n in zip(first, lens)],
                hq, dt, 50, rope, ps)
    for again in range(2):                                      # the second writes the same rows
        q, want = _append(cache, oracle, tables, starts, counts, hq, dt, 60, rope, ps, left=2)
        assert torch.equal(q, want)
        _assert_cache(cache, oracle, tables, lens)
    untouched = np.setdiff1d(np.arange(pages), np.concatenate(tables))
    for t, b in zip(cache, before):
        assert torch.equal(t.view(torch.uint8)[untouched], b.view(torch.uint8)[untouched])


@pytest.mark.parametrize("dt,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_append_token_by_token_grows_the_scale(dt, d):
    """Tokens of growing size, one a call: every step re-rounds the page's older codes."""
    cache, oracle = ops.kv8_pages(6, 16, 2, d, DEV), kv8.Cache(6, 2, 16, d)
    table = [np.array([4, 2, 5], np.int32)]
    for t in range(40):
        q, want = _append(cache, oracle, table, [t], [1], 4, dt, 7 * t, True, 16, spread=2.0)
        assert torch.equal(q, want)
        _assert_cache(cache, oracle, table, [t + 1])


@pytest.mark.parametrize("n", [1, 20])
def test_append_zeros_and_values_that_are_not_finite(n):
    hkv, d = 2, 64
    cache = ops.kv8_pages(4, 16, hkv, d, DEV)
    k = torch.zeros(n, hkv, d, dtype=torch.bfloat16)
    v = U.rows((n, hkv, d), torch.bfloat16, 3)
    v[0, 1, 5] = math.inf
    ptr, idx, lpl = U.csr([np.array([1, 3], np.int32)[:-(-n // 16)]], [n], 16, DEV)
    qo = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    ops.rope_kv8_append(None, k.to(DEV), v.to(DEV), None, None, *cache, qo, n, ptr, idx, lpl,
                        rotate=False)
    sk, sv = cache[2].cpu(), cache[3].cpu()
    assert bool((sk[1] == 0).all()) and bool(torch.isnan(sv[1, 1])) and bool(sv[1, 0] > 0)
    kk, vv = ops.kv8_gather(*cache, ptr, idx, lpl, torch.bfloat16)
    assert bool((kk == 0).all())
    assert bool(torch.isnan(vv[0, :min(n, 16), 1]).all()) and bool(torch.isfinite(vv[0, :, 0]).all())
    if n > 16:
        assert bool(torch.isfinite(vv[1]).all())
    # the block stays NaN while its page lasts, and a page begun again is clean
    if n == 1:
        ptr2, idx2, lpl2 = U.csr([np.array([1], np.int32)], [2], 16, DEV)
        one = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
        fine = U.rows((1, hkv, d), torch.bfloat16, 4).to(DEV)
        ops.rope_kv8_append(None, fine, fine, None, None, *cache, one, 1, ptr2, idx2, lpl2, rotate=False)
        assert bool(torch.isnan(cache[3][1, 1]))
        ops.rope_kv8_append(None, fine, fine, None, None, *cache, one, 1, ptr, idx, lpl, rotate=False)
        assert bool(torch.isfinite(cache[3][1]).all())


@pytest.mark.parametrize("dt,d,ps", [(torch.bfloat16, 128, 16), (torch.float16, 64, 16), (torch.float32, 64, 16),
                                     (torch.bfloat16, 96, 5)])
@pytest.mark.parametrize("first", [1, 3])
@pytest.mark.parametrize("stale", [math.nan, 2.0 ** 20])
def test_a_page_begun_with_zeros_forgets_its_last_owner(dt, d, ps, first, stale):
    """Head rows of zeros in the first slots of a page whose scales are left over, alone in their
    call and together; then small tokens one by one."""
    hkv, page = 2, 3
    cache = U.random_cache(5, hkv, ps, d, DEV, 7)
    cache[2].fill_(stale)
    cache[3].fill_(stale)
    oracle = kv8.Cache(5, hkv, ps, d)
    table = [np.array([page], np.int32)]
    start = 0
    for count in (first, 1, 1):
        k = torch.zeros(count, hkv, d, dtype=dt) if start == 0 else U.rows((count, hkv, d), dt, start) / 16
        v = k.clone()
        k[:, 1] = U.rows((count, d), dt, 9)                  # the other kv head has values from the start
        ptr, idx, lpl = U.csr(table, [start + count], ps, DEV)
        qo = torch.tensor([0, count], dtype=torch.int32, device=DEV)
        ops.rope_kv8_append(None, k.to(DEV), v.to(DEV), None, None, *cache, qo, count, ptr, idx, lpl, rotate=False)
        oracle.append(table[0], start, k.float().numpy(), v.float().numpy())
        start += count
        _assert_cache(cache, oracle, table, [start])


def test_append_bad_plans_are_reported_and_skipped():
    hkv, d = 2, 64
    cache = U.random_cache(8, hkv, 16, d, DEV, 5)
    before = [t.clone() for t in cache]
    x = U.rows((12, hkv, d), torch.bfloat16, 1).to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(64, d))

    def run(qo, most, table, length, rows=None, tables=(cos, sin), last=None):
        ptr, idx, lpl = U.csr([np.array(table, np.int32)], [length], 16, DEV)
        if last is not None:
            lpl.fill_(last)
        rs = None if rows is None else torch.tensor([rows], dtype=torch.int32, device=DEV)
        q = torch.full_like(x, 9.0)
        ops.rope_kv8_append(x, x, x, *tables, *cache, torch.tensor([0, qo], dtype=torch.int32, device=DEV),
                            most, ptr, idx, lpl, q_row_start=rs, q_out=q)
        return q

    for args, what in (((12, 12, [1], 5), "plan entry"), ((12, 4, [1], 16), "plan entry"),
                       ((4, 4, [1], 16, 10), "plan entry"), ((4, 4, [1], 16, -1), "plan entry"),
                       ((1, 1, [1], 16, None, (cos, sin), 17), "plan entry"),
                       ((4, 4, [1], 16, None, (cos, sin), 0), "plan entry"),
                       ((4, 4, [8], 16), "page id"), ((4, 4, [-1], 16), "page id")):
        q = run(*args)
        with pytest.raises(RuntimeError, match=what):
            ops.check_device_status(DEV)
        assert what == "page id" or bool((q == 9.0).all())
        for t, b in zip(cache, before):
            assert torch.equal(t.view(torch.uint8), b.view(torch.uint8))
    run(4, 4, [1], 16, None, (cos[:14].contiguous(), sin[:14].contiguous()))   # positions 12 to 15
    with pytest.raises(RuntimeError, match="RoPE table"):
        ops.check_device_status(DEV)


@pytest.mark.parametrize("dt,hq,hkv,d,ps", [(torch.bfloat16, 32, 8, 128, 16), (torch.float16, 12, 2, 64, 16),
                                            (torch.float32, 4, 2, 64, 16), (torch.bfloat16, 6, 3, 96, 5)])
@pytest.mark.parametrize("counts", [[1, 1, 1], [40, 3, 1]])
def test_append_turns_q_in_place(dt, hq, hkv, d, ps, counts):
    lens = [n + s for n, s in zip(counts, (7, 0, 30))]
    tables = U.page_lists(lens, ps, 40, 4)
    cos, sin = (t.to(DEV) for t in _tables(max(lens), d))
    plan = U.csr(tables, lens, ps, DEV)
    qo = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=DEV)
    q, k, v = (U.rows((sum(counts), h, d), dt, 5 + h).to(DEV) for h in (hq, hkv, hkv))
    first, second = (U.random_cache(40, hkv, ps, d, DEV, 6) for _ in range(2))
    want = ops.rope_kv8_append(q, k, v, cos, sin, *first, qo, max(counts), *plan)
    assert not torch.equal(want, q)
    assert ops.rope_kv8_append(q, k, v, cos, sin, *second, qo, max(counts), *plan, q_out=q) is q
    assert torch.equal(q, want)
    for a, b in zip(first, second):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hkv,d,ps,lens", [(8, 128, 16, [1, 0, 33, 512]), (2, 64, 16, [300]),
                                           (3, 96, 5, [7, 5, 1]), (1, 256, 64, [65])])
def test_gather_is_code_times_scale(dt, hkv, d, ps, lens):
    pages = sum(-(-n // ps) for n in lens) + 3
    tables = U.page_lists(lens, ps, pages, 3)
    cache = U.random_cache(pages, hkv, ps, d, DEV, 4, power=False)
    cache[0].view(torch.uint8)[:, :, ps - 1, 0] = 0x7F          # NaN codes, kept where in length
    ptr, idx, lpl = U.csr(tables, lens, ps, DEV, spare=2)
    total = sum(len(t) for t in tables)
    out = tuple(torch.full((total + 2, ps, hkv, d), 7.0, dtype=dt, device=DEV) for _ in range(2))
    got = ops.kv8_gather(*cache, ptr, idx, lpl, dt, out=out)
    for i in range(2):
        assert got[i] is out[i]
        at = 0
        for t, n in zip(tables, lens):
            x = got[i][at:at + len(t)].cpu().reshape(-1, hkv, d)
            # one product of a code and a scale, rounded to fp32 and once to dt
            want = torch.from_numpy(U.values(cache[i], cache[2 + i], t, n)).float().to(dt)
            torch.testing.assert_close(x[:n], want, rtol=0, atol=0, equal_nan=True)
            assert bool((x[n:] == 0).all())
            at += len(t)
        assert bool((got[i][total:] == 7.0).all())


def test_gather_saturates_finite_values_to_fp16():
    cache = ops.kv8_pages(2, 16, 1, 32, DEV)
    x = torch.full((1, 1, 32), 65504.0, dtype=torch.float16, device=DEV)
    ptr, idx, lpl = U.csr([np.array([1], np.int32)], [1], 16, DEV)
    qo = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    ops.rope_kv8_append(None, x, -x, None, None, *cache, qo, 1, ptr, idx, lpl, rotate=False)
    k, v = ops.kv8_gather(*cache, ptr, idx, lpl, torch.float16)
    assert bool((k[0, 0] == 65504.0).all()) and bool((v[0, 0] == -65504.0).all())
    k32, _ = ops.kv8_gather(*cache, ptr, idx, lpl, torch.float32)
    assert bool((k32[0, 0] == 65536.0).all())


def _check_attention(out, q, cache, tables, lens, counts, row_start, sm_scale, p_half, causal=True,
                     more=0.0):
    out = out.cpu()
    for b, (t, n, c) in enumerate(zip(tables, lens, counts)):
        r = slice(row_start[b], row_start[b] + c)
        k, v = (U.values(cache[i], cache[2 + i], t, n) for i in range(2))
        qd = q[r].cpu().double().numpy()
        want = kv8.attention(qd, k, v, sm_scale, causal)
        vs = U.token_scales(cache[3], t, n, cache[0].shape[2])
        bound = U.attention_bound(qd, k, v, vs, sm_scale, want, out.dtype, p_half, causal) + more
        got = out[r].double().numpy()
        # an exact value that the bound takes past the type's largest one (fp16: 65504; from
        # 65520 on the nearest value is an infinity) may be the infinity of its sign
        most = torch.finfo(out.dtype).max
        past = (np.abs(want) + bound > most) & np.isinf(got) & (np.sign(got) == np.sign(want))
        err = np.where(past, 0.0, np.abs(got - want))
        assert not np.isnan(err).any(), (b, n)
        assert (err <= bound).all(), (b, n, float((err / bound).max()))


DECODE = [
    # dtype, hq, hkv, d, page size, lens
    (torch.bfloat16, 32, 8, 128, 16, [1, 15, 16, 17, 100, 1000]),
    (torch.float16, 32, 8, 128, 16, [513]),
    (torch.float16, 16, 2, 128, 16, [0, 33, 0, 700, 0]),
    (torch.bfloat16, 4, 1, 128, 16, [2, 31, 32, 600]),
    (torch.bfloat16, 16, 1, 128, 16, [77, 1200]),
    (torch.bfloat16, 64, 8, 128, 16, [40, 513]),
    (torch.float16, 8, 8, 128, 16, [19, 260]),
    (torch.bfloat16, 8, 2, 64, 16, [9, 300, 1024]),
    (torch.float16, 12, 3, 64, 16, [5, 160, 64]),
    (torch.bfloat16, 10, 5, 128, 16, [129, 48, 3]),
    (torch.bfloat16, 34, 2, 128, 16, [70, 5]),
    (torch.float32, 4, 2, 64, 16, [1, 50, 33]),
    (torch.float32, 32, 8, 128, 16, [130]),
    (torch.bfloat16, 6, 3, 96, 5, [12, 1]),
    (torch.float16, 2, 1, 256, 64, [65]),
]


def _p_half(dt):
    # the products of 16-bit types take probabilities of the type or of fp16
    return U.HALF[dt] if dt != torch.float32 else 0.0


@pytest.mark.parametrize("dt,hq,hkv,d,ps,lens", DECODE)
def test_decode_is_the_definition(dt, hq, hkv, d, ps, lens):
    pages = sum(-(-n // ps) for n in lens) + 3
    tables = U.page_lists(lens, ps, pages, 11)
    cache = U.random_cache(pages, hkv, ps, d, DEV, 12, power=d != 64)
    for t, n in zip(tables, lens):
        if n % ps:                                  # slots behind the last token hold NaN codes
            for pool in cache[:2]:
                pool.view(torch.uint8)[int(t[-1]), :, n % ps:] = 0x7F
    wide = U.rows((len(lens), hq + 2, d), dt, 13).to(DEV)
    q = wide[:, 1:-1]                               # a strided view
    sm = 1 / math.sqrt(d)
    plan = U.csr(tables, lens, ps, DEV, spare=1)
    out = ops.paged_decode_kv8(q, *cache, *plan, sm)
    _check_attention(out, q, cache, tables, lens, [1] * len(lens), list(range(len(lens))), sm,
                     _p_half(dt))
    again = torch.full((len(lens), hq + 1, d), 3.0, dtype=dt, device=DEV)
    ops.paged_decode_kv8(q, *cache, *plan, sm, out=again[:, :hq])
    assert torch.equal(again[:, :hq], out) and bool((again[:, hq] == 3.0).all())


PREFILL = [
    # dtype, hq, hkv, d, page size, lens, new rows, causal, left padding
    (torch.bfloat16, 32, 8, 128, 16, [33, 17, 64], [33, 1, 20], True, 0),
    (torch.bfloat16, 32, 8, 128, 16, [300], [5], True, 0),
    (torch.float16, 32, 8, 128, 16, [700, 40, 0], [3, 4, 0], True, 3),
    (torch.float16, 8, 2, 128, 16, [100, 260], [100, 130], True, 0),
    (torch.bfloat16, 8, 8, 128, 16, [65, 10], [60, 10], False, 1),
    (torch.bfloat16, 4, 2, 64, 16, [50, 31], [50, 2], True, 0),
    (torch.float16, 16, 2, 64, 16, [129], [100], True, 2),
    (torch.float16, 12, 2, 128, 16, [40], [12], True, 0),
    (torch.bfloat16, 34, 2, 128, 16, [20], [6], True, 0),
    (torch.bfloat16, 64, 4, 128, 16, [300, 77], [300, 40], True, 0),
    (torch.float16, 4, 4, 128, 16, [700], [260], True, 0),
    (torch.bfloat16, 8, 2, 128, 16, [513, 128, 129, 1], [70, 128, 129, 1], False, 0),
    (torch.bfloat16, 16, 8, 128, 16, [256, 127, 384], [256, 127, 300], True, 5),
    # more work items than SMs
    (torch.bfloat16, 16, 4, 128, 16, [170 + 9 * i for i in range(24)], [150 + 5 * i for i in range(24)], True, 0),
    (torch.float16, 8, 8, 128, 16, [400 - 9 * i for i in range(20)], [300 - 9 * i for i in range(20)], True, 0),
    (torch.bfloat16, 8, 2, 64, 16, [400 - 9 * i for i in range(20)], [300 - 9 * i for i in range(20)], True, 0),
    (torch.float16, 6, 6, 64, 16, [63, 64, 65, 1, 200], [63, 64, 65, 1, 200], False, 2),
    (torch.bfloat16, 16, 1, 64, 16, [17, 130, 33], [17, 9, 33], True, 1),
    (torch.float16, 16, 8, 64, 16, [70, 530], [70, 290], True, 0),
    (torch.float32, 4, 2, 64, 16, [32, 20], [32, 1], True, 0),
    (torch.bfloat16, 6, 3, 96, 5, [12, 6], [5, 6], True, 1),
]


def _with_idle(cases, shape):
    """Each case as it is and, where it would take another kernel then, in a batch made large
    by sequences without rows; ``shape``: (dtype, batch, hq, hkv, max_qo_len, page size)."""
    out = []
    for case in cases:
        dt, batch, hq, hkv, new, ps = shape(case)
        out.append((*case, 0))
        idle = U.idle_for_tiles(batch, hq, hkv, new)
        if dt != torch.float32 and ps == 16 and idle and 128 % (hq // hkv) == 0:
            out.append((*case, idle))
    return out


@pytest.mark.parametrize("dt,hq,hkv,d,ps,lens,counts,causal,left,idle", _with_idle(
    PREFILL, lambda c: (c[0], len(c[5]), c[1], c[2], max(c[6]), c[4])))
def test_prefill_is_the_definition(dt, hq, hkv, d, ps, lens, counts, causal, left, idle):
    lens, counts = lens + [0] * idle, counts + [0] * idle
    pages = sum(-(-n // ps) for n in lens) + 3
    tables = U.page_lists(lens, ps, pages, 21)
    cache = U.random_cache(pages, hkv, ps, d, DEV, 22)
    for t, n in zip(tables, lens):
        if n % ps:
            for pool in cache[:2]:
                pool.view(torch.uint8)[int(t[-1]), :, n % ps:] = 0x7F
    width = max(counts) + left
    row_start = ([b * width + width - c for b, c in enumerate(counts)] if left
                 else [int(x) for x in np.cumsum([0] + counts)[:-1]])
    nrows = len(lens) * width if left else sum(counts)
    q = U.rows((nrows, hq, d), dt, 23).to(DEV)
    out = torch.full_like(q, 5.0)
    sm = 1 / math.sqrt(d)
    plan = U.csr(tables, lens, ps, DEV, spare=1)
    qo = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=DEV)
    rs = torch.tensor(row_start, dtype=torch.int32, device=DEV) if left else None
    ops.paged_prefill_kv8(q, qo, max(counts), *cache, *plan, sm, causal=causal, q_row_start=rs, out=out)
    _check_attention(out, q, cache, tables, lens, counts, row_start, sm, _p_half(dt), causal)
    real = torch.zeros(nrows, dtype=torch.bool)
    for s, c in zip(row_start, counts):
        real[s:s + c] = True
    assert bool((out[~real.to(DEV)] == 5.0).all())


@pytest.mark.parametrize("dt,d,idle", [(torch.bfloat16, 128, 0), (torch.float16, 64, 0), (torch.float32, 64, 0),
                                       (torch.bfloat16, 128, 90), (torch.float16, 64, 90)])
def test_prefill_rows_that_see_nothing_are_zeros(dt, d, idle):
    """More rows than positions (row i sits at kv_len - qo_len + i < 0), and rows of a
    sequence without pages."""
    hq, hkv, ps = 8, 2, 16
    cache = U.random_cache(8, hkv, ps, d, DEV, 2)
    lens, counts = [3, 0, 20] + [0] * idle, [5, 4, 2] + [0] * idle
    if idle:                                        # and a second pair of tiles of such rows
        lens[1], counts[1] = 0, 80
        lens[2], counts[2] = 20, 150
    tables = U.page_lists(lens, ps, 8, 1)
    q = U.rows((sum(counts), hq, d), dt, 3).to(DEV)
    qo = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 5.0)
    sm = 1 / math.sqrt(d)
    ops.paged_prefill_kv8(q, qo, max(counts), *cache, *U.csr(tables, lens, ps, DEV), sm, out=out)
    starts = [int(x) for x in np.cumsum([0] + counts)[:-1]]
    _check_attention(out, q, cache, tables, lens, counts, starts, sm, _p_half(dt))
    assert bool((out[:2] == 0).all()) and bool((out[5:5 + counts[1]] == 0).all())


@pytest.mark.parametrize("dt,d,rows,idle", _with_idle(
    [(torch.bfloat16, 128, 1), (torch.float16, 64, 7), (torch.bfloat16, 128, 90), (torch.float16, 128, 150),
     (torch.float16, 64, 90), (torch.float32, 64, 5)], lambda c: (c[0], 1, 8, 2, c[2], 16)))
def test_scales_of_neighbouring_pages_may_differ_by_any_factor(dt, d, rows, idle):
    """V scales over 40 powers of two, K scales over 8 (zeros and non-powers among them): the
    pages with the large values get next to no weight where K is large."""
    hq, hkv, n = 8, 2, 333
    cache = U.random_cache(30, hkv, 16, d, DEV, 31)
    table = U.page_lists([n], 16, 30, 32)
    g = torch.Generator().manual_seed(33)
    for t, lo, hi in ((cache[2], -11, -3), (cache[3], -20, 20)):
        s = torch.exp2(torch.randint(lo, hi, t.shape, generator=g).float())
        s[torch.rand(t.shape, generator=g) < 0.15] = 0.0
        s[int(table[0][3])] = 0.0
        s[:, 1] *= 1.0 + torch.rand(t.shape[0], generator=g)
        t.copy_(s)
    q = (U.rows((rows, hq, d), dt, 34) * 2).to(DEV)
    sm = 1 / math.sqrt(d)
    lens, tables = [n] + [0] * idle, table + [table[0][:0]] * idle
    plan = U.csr(tables, lens, 16, DEV)
    qo = torch.tensor([0] + [rows] * (1 + idle), dtype=torch.int32, device=DEV)
    out = ops.paged_prefill_kv8(q, qo, rows, *cache, *plan, sm)
    _check_attention(out, q, cache, table, [n], [rows], [0], sm, _p_half(dt))
    if rows == 1:
        out = ops.paged_decode_kv8(q, *cache, *plan, sm)
        _check_attention(out, q, cache, table, [n], [1], [0], sm, _p_half(dt))


@pytest.mark.parametrize("lo,hi", [(-98, -90), (96, 104)])
@pytest.mark.parametrize("d,rows,idle", _with_idle([(128, 1), (128, 40), (64, 40)],
                                                   lambda c: (torch.bfloat16, 1, 8, 2, c[1], 16)))
def test_scales_far_from_one(d, rows, idle, lo, hi):
    """V scales whose inverses, summed over a row, come near fp32's limits."""
    hq, hkv, n = 8, 2, 200
    cache = U.random_cache(20, hkv, 16, d, DEV, 51)
    table = U.page_lists([n], 16, 20, 52)
    g = torch.Generator().manual_seed(53)
    cache[3].copy_(torch.exp2(torch.randint(lo, hi, cache[3].shape, generator=g).float()))
    q = U.rows((rows, hq, d), torch.bfloat16, 54).to(DEV)
    plan = U.csr(table + [table[0][:0]] * idle, [n] + [0] * idle, 16, DEV)
    qo = torch.tensor([0] + [rows] * (1 + idle), dtype=torch.int32, device=DEV)
    sm = 1 / math.sqrt(d)
    out = ops.paged_prefill_kv8(q, qo, rows, *cache, *plan, sm)
    _check_attention(out, q, cache, table, [n], [rows], [0], sm, _p_half(torch.bfloat16))


@pytest.mark.parametrize("dt,d,rows,idle", _with_idle(
    [(torch.bfloat16, 128, 1), (torch.float16, 128, 9), (torch.bfloat16, 64, 40), (torch.float16, 128, 90)],
    lambda c: (c[0], 1, 8, 2, c[2], 16)))
@pytest.mark.parametrize("seed", range(6))
def test_zero_v_blocks_beside_large_scores(dt, d, rows, idle, seed):
    """Scores up to some hundreds, the largest often on blocks of zeros in V: before the first
    block that has values, between such blocks, and far above or below them.

    On top of attention_bound: a weight that the kernels hold in fp16 is off by at most 2^-25
    beside M. Where a block of zeros has set M, that is 2^-60 of the zeros' weight times the
    scale of blocks before it, or 2^-90 of it before any: the row's sum is at least the zeros'
    weight, so 2^-85 scale_v + 2^-115 times the sum of the codes."""
    hq, hkv, n = 8, 2, 420
    pages = -(-n // 16)
    cache = U.random_cache(pages + 2, hkv, 16, d, DEV, 100 + seed)
    table = U.page_lists([n], 16, pages + 2, 200 + seed)
    g = torch.Generator().manual_seed(300 + seed)
    at = torch.from_numpy(table[0]).long()
    zero = torch.rand(pages, hkv, generator=g) < 0.4
    zero[:seed] = True                              # leading ones
    scale = torch.exp2(torch.randint(-12, 0, (pages, hkv), generator=g).float())
    scale[zero] = 0.0
    cache[3][at.to(DEV)] = scale.to(DEV)
    cache[2][at.to(DEV)] = torch.exp2(torch.randint(-6, 0, (pages, hkv), generator=g).float()).to(DEV)
    q = U.rows((rows, hq, d), dt, 400 + seed).to(DEV)
    lens, tables = [n] + [0] * idle, table + [table[0][:0]] * idle
    qo = torch.tensor([0] + [rows] * (1 + idle), dtype=torch.int32, device=DEV)
    sm = 1 / math.sqrt(d)
    out = ops.paged_prefill_kv8(q, qo, rows, *cache, *U.csr(tables, lens, 16, DEV), sm)
    codes = U.values(cache[1], torch.ones_like(cache[3]), table[0], n)
    sums = np.repeat(np.abs(codes).sum(0), hq // hkv, 0)[None]
    most = np.repeat(scale.double().numpy().max(0), hq // hkv)[None, :, None]
    _check_attention(out, q, cache, table, [n], [rows], [0], sm, _p_half(dt),
                     more=(2.0 ** -85 * most + 2.0 ** -115) * sums)


def test_v_blocks_of_the_smallest_scales():
    """Scales of 2^-126 .. 2^-101: the outputs are at most the values themselves, never
    infinite or NaN, and a larger block beside them is exact."""
    hq, hkv, d, n = 8, 2, 128, 96
    for rows, idle in ((1, 0), (40, U.idle_for_tiles(1, hq, hkv, 40))):
        cache = U.random_cache(8, hkv, 16, d, DEV, 61)
        table = U.page_lists([n], 16, 8, 62)
        cache[3].copy_(torch.exp2(torch.randint(-126, -100, cache[3].shape,
                                                generator=torch.Generator().manual_seed(63)).float()))
        q = U.rows((rows, hq, d), torch.bfloat16, 64).to(DEV)
        plan = U.csr(table + [table[0][:0]] * idle, [n] + [0] * idle, 16, DEV)
        qo = torch.tensor([0] + [rows] * (1 + idle), dtype=torch.int32, device=DEV)
        out = ops.paged_prefill_kv8(q, qo, rows, *cache, *plan, 0.1).float()
        assert bool((out.abs() <= 448 * 2.0 ** -100).all())
        cache[3][int(table[0][2])] = 0.5
        out = ops.paged_prefill_kv8(q, qo, rows, *cache, *plan, 0.1)
        _check_attention(out, q, cache, table, [n], [rows], [0], 0.1, _p_half(torch.bfloat16))


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("dt,rows,idle", _with_idle(
    [(torch.bfloat16, 12), (torch.float16, 150), (torch.bfloat16, 260), (torch.float32, 40)],
    lambda c: (c[0], 1, 8, 2, c[1], 16)))
def test_a_block_that_is_not_finite_in_a_masked_place(dt, rows, idle, which):
    """Rows that come before the block see nothing of it; the others are NaN."""
    hq, hkv, d, n = 8, 2, 128, 300
    cache = U.random_cache(22, hkv, 16, d, DEV, 41)
    table = U.page_lists([n], 16, 22, 42)
    bad = n // 16 - 0                                # the last, partly filled page
    page = int(table[0][bad])
    i = "kv".index(which)
    cache[2 + i][page, 1] = math.nan
    cache[i].view(torch.uint8)[page, 1] = 0          # as the append leaves such a block
    q = U.rows((rows, hq, d), dt, 43).to(DEV)
    sm = 1 / math.sqrt(d)
    plan = U.csr(table + [table[0][:0]] * idle, [n] + [0] * idle, 16, DEV)
    qo = torch.tensor([0] + [rows] * (1 + idle), dtype=torch.int32, device=DEV)
    out = ops.paged_prefill_kv8(q, qo, rows, *cache, *plan, sm).cpu()
    first = bad * 16 - (n - rows)                    # first row that sees the block
    assert 0 <= first < rows or rows == 12
    first = max(first, 0)
    assert bool(torch.isnan(out[first:, 4:]).all())
    assert bool(torch.isfinite(out[:first]).all()) and bool(torch.isfinite(out[:, :4]).all())


def test_attention_bad_pages_are_reported():
    hq, hkv, d = 8, 2, 128
    for dt in (torch.bfloat16, torch.float32):
        cache = U.random_cache(4, hkv, 16, d, DEV, 2)
        q = U.rows((3, hq, d), dt, 3).to(DEV)
        ptr, idx, lpl = U.csr([np.array([1, 99], np.int32)], [20], 16, DEV)
        ops.paged_decode_kv8(q[:1], *cache, ptr, idx, lpl, 0.1)
        with pytest.raises(RuntimeError, match="page id"):
            ops.check_device_status(DEV)
        qo = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
        ops.paged_prefill_kv8(q, qo, 3, *cache, ptr, idx, lpl, 0.1)
        with pytest.raises(RuntimeError, match="page id"):
            ops.check_device_status(DEV)
        if dt != torch.float32:                     # the kernel of the large batches
            idle = U.idle_for_tiles(1, hq, hkv, 20)
            q20 = U.rows((20, hq, d), dt, 3).to(DEV)
            big = U.csr([np.array([1, 99], np.int32)] + [np.zeros(0, np.int32)] * idle, [20] + [0] * idle, 16, DEV)
            qo = torch.tensor([0] + [20] * (1 + idle), dtype=torch.int32, device=DEV)
            out = ops.paged_prefill_kv8(q20, qo, 20, *cache, *big, 0.1)
            with pytest.raises(RuntimeError, match="page id"):
                ops.check_device_status(DEV)
            assert bool(torch.isfinite(out).all())
        ops.kv8_gather(*cache, ptr, idx, lpl, dt)
        with pytest.raises(RuntimeError, match="page id"):
            ops.check_device_status(DEV)


@pytest.mark.parametrize("dt,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("rows,idle", [(1, 0), (3, 0), (20, True)])
@pytest.mark.parametrize("bad", [99, -1, 4])
def test_rows_that_see_a_bad_page_are_finite(dt, d, rows, idle, bad):
    """Whatever page 0 holds: NaN codes, NaN scales."""
    hq, hkv = 8, 2
    cache = U.random_cache(4, hkv, 16, d, DEV, 2)
    for t in cache[:2]:
        t.view(torch.uint8)[0] = 0x7F
    for t in cache[2:]:
        t[0] = math.nan
    idle = U.idle_for_tiles(1, hq, hkv, rows) if idle else 0
    none = [np.zeros(0, np.int32)] * idle
    plan = U.csr([np.array([1, bad, 2], np.int32)] + none, [40] + [0] * idle, 16, DEV)
    q = U.rows((rows, hq, d), dt, 3).to(DEV)
    qo = torch.tensor([0] + [rows] * (1 + idle), dtype=torch.int32, device=DEV)
    outs = [ops.paged_prefill_kv8(q, qo, rows, *cache, *plan, 0.1)]
    if rows == 1:
        outs.append(ops.paged_decode_kv8(q, *cache, *plan, 0.1))
    with pytest.raises(RuntimeError, match="page id"):
        ops.check_device_status(DEV)
    for out in outs:
        assert bool(torch.isfinite(out).all())


def test_a_block_that_is_not_finite_reads_as_nan():
    hq, hkv, d = 8, 2, 128
    for dt in (torch.bfloat16, torch.float32):
        cache = U.random_cache(4, hkv, 16, d, DEV, 2)
        plan = U.csr([np.array([1, 2], np.int32)], [30], 16, DEV)
        q = U.rows((1, hq, d), dt, 3).to(DEV)
        for i in (2, 3):
            keep = cache[i][2, 1].clone()
            cache[i][2, 1] = math.nan
            out = ops.paged_decode_kv8(q, *cache, *plan, 0.1)
            assert bool(torch.isnan(out[0, 4:]).all()) and bool(torch.isfinite(out[0, :4]).all())
            cache[i][2, 1] = keep


def test_bad_last_page_lengths_are_reported():
    hq, hkv, d = 8, 2, 128
    for dt, rows in ((torch.bfloat16, 1), (torch.bfloat16, 20), (torch.float32, 3)):
        cache = U.random_cache(4, hkv, 16, d, DEV, 2)
        idle = U.idle_for_tiles(1, hq, hkv, rows) if rows == 20 else 0
        ptr, idx, lpl = U.csr([np.array([1, 2], np.int32)] + [np.zeros(0, np.int32)] * idle,
                              [30] + [0] * idle, 16, DEV)
        q = U.rows((rows, hq, d), dt, 3).to(DEV)
        qo = torch.tensor([0] + [rows] * (1 + idle), dtype=torch.int32, device=DEV)
        for last in (0, 17, 2 ** 31 - 1, -2 ** 31):
            lpl[0] = last
            ops.paged_prefill_kv8(q, qo, rows, *cache, ptr, idx, lpl, 0.1)
            with pytest.raises(RuntimeError, match="plan entry"):
                ops.check_device_status(DEV)


def test_more_sequences_than_shared_memory_holds():
    """The page list's bounds are read from global memory behind 2048 sequences."""
    hq, hkv, d, n = 2, 1, 64, 2100
    lens = [(7 * i) % 41 for i in range(n)]
    pages = sum(-(-x // 16) for x in lens) + 1
    tables = U.page_lists(lens, 16, pages, 71)
    cache = U.random_cache(pages, hkv, 16, d, DEV, 72)
    q = U.rows((n, hq, d), torch.bfloat16, 73).to(DEV)
    out = ops.paged_decode_kv8(q, *cache, *U.csr(tables, lens, 16, DEV), 0.125)
    _check_attention(out, q, cache, tables, lens, [1] * n, list(range(n)), 0.125, U.HALF[torch.bfloat16])


def test_max_qo_len_beyond_the_rows():
    """A bound above the rows there are changes nothing, however large."""
    hq, hkv, d, lens, counts = 16, 2, 64, [40, 9], [3, 2]
    cache = U.random_cache(8, hkv, 16, d, DEV, 81)
    tables = U.page_lists(lens, 16, 8, 82)
    plan = U.csr(tables, lens, 16, DEV)
    q = U.rows((5, hq, d), torch.bfloat16, 83).to(DEV)
    qo = torch.tensor([0, 3, 5], dtype=torch.int32, device=DEV)
    out = ops.paged_prefill_kv8(q, qo, 2 ** 31 - 1, *cache, *plan, 0.125)
    _check_attention(out, q, cache, tables, lens, counts, [0, 3], 0.125, U.HALF[torch.bfloat16])
    k = U.rows((5, hkv, d), torch.bfloat16, 84).to(DEV)
    got, want = ([t.clone() for t in cache] for _ in range(2))
    ops.rope_kv8_append(None, k, k, None, None, *got, qo, 2 ** 31 - 1, *plan, rotate=False)
    ops.rope_kv8_append(None, k, k, None, None, *want, qo, 3, *plan, rotate=False)
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dt,hq,hkv,d,ps", [(torch.bfloat16, 32, 8, 128, 16), (torch.float16, 6, 2, 64, 16),
                                            (torch.float32, 4, 2, 64, 16), (torch.bfloat16, 6, 3, 96, 5)])
@pytest.mark.parametrize("first,last", [(2, 6), (5, 6), (0, 3), (3, 3)])
def test_a_part_of_a_longer_batch(dt, hq, hkv, d, ps, first, last):
    """Bounds sliced out of a batch of seven, over its whole list: the results of the sequences'
    own list."""
    lens, counts = [60, 900, 33, 0, 700, 18, 45], [7, 5, 1, 0, 6, 2, 3]
    pages = sum(-(-n // ps) for n in lens) + 1
    tables = U.page_lists(lens, ps, pages, 61)
    caches = [U.random_cache(pages, hkv, ps, d, DEV, 62) for _ in range(2)]
    ptr, idx, lpl = U.csr(tables, lens, ps, DEV)
    part = (ptr[first:last + 1], idx, lpl[first:last])
    own = U.csr(tables[first:last], lens[first:last], ps, DEV)
    q = U.rows((sum(counts), hq, d), dt, 63).to(DEV)
    k = U.rows((sum(counts), hkv, d), dt, 64).to(DEV)
    qo = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=DEV)[first:last + 1]
    r0, r1 = int(sum(counts[:first])), int(sum(counts[:last]))
    got = []
    for cache, plan in zip(caches, (part, own)):
        ops.rope_kv8_append(None, k, -k, None, None, *cache, qo, 7, *plan, rotate=False)
        out = torch.full_like(q, 3.0)
        ops.paged_prefill_kv8(q, qo, 7, *cache, *plan, 0.1, out=out)
        dec = ops.paged_decode_kv8(q[:last - first], *cache, *plan, 0.1)
        at = int(ptr[first]) if plan is part else 0
        n = int(ptr[last] - ptr[first])
        back = tuple(torch.full((plan[1].numel(), ps, hkv, d), 7.0, dtype=dt, device=DEV) for _ in range(2))
        ops.kv8_gather(*cache, *plan, dt, out=back)
        for t in back:
            assert bool((t[:at] == 7.0).all()) and bool((t[at + n:] == 7.0).all())
        assert bool((out[:r0] == 3.0).all()) and bool((out[r1:] == 3.0).all())
        got.append([out, dec, *(t[at:at + n] for t in back), *(t.view(torch.uint8) for t in cache)])
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """The same pages at the end of a pool of 2^32 bytes and more a tensor."""
    hq, hkv, d, lens, counts = 32, 8, 128, [70, 33, 200], [20, 1, 45]
    few = sum(-(-n // 16) for n in lens) + 1
    small = U.random_cache(few, hkv, 16, d, DEV, 91)
    far = 2 ** 32 // (hkv * 16 * d) + 1
    big = ops.kv8_pages(far + few, 16, hkv, d, DEV)
    for b, s in zip(big, small):
        b[far:].view(torch.uint8).copy_(s.view(torch.uint8))
    tables = U.page_lists(lens, 16, few, 92)
    ptr, idx, lpl = U.csr(tables, lens, 16, DEV)
    q = U.rows((sum(counts), hq, d), torch.bfloat16, 93).to(DEV)
    k = U.rows((sum(counts), hkv, d), torch.bfloat16, 94).to(DEV)
    qo = torch.tensor(np.cumsum([0] + counts), dtype=torch.int32, device=DEV)
    idle = U.idle_for_tiles(3, hq, hkv, 45)
    results = []
    for cache, at in ((small, 0), (big, far)):
        plan = (ptr, idx + at, lpl)
        ops.rope_kv8_append(None, k, -k, None, None, *cache, qo, 45, *plan, rotate=False)
        one = (q[:3].contiguous(), *cache, *plan, 0.1)
        wide = (torch.cat([ptr, ptr[-1:].expand(idle)]), idx + at, torch.cat([lpl, lpl[:1].expand(idle)]))
        qo_wide = torch.cat([qo, qo[-1:].expand(idle)])
        results.append([*ops.kv8_gather(*cache, *plan, torch.bfloat16), ops.paged_decode_kv8(*one),
                        ops.paged_prefill_kv8(q, qo, 45, *cache, *plan, 0.1),
                        ops.paged_prefill_kv8(q, qo_wide, 45, *cache, *wide, 0.1)])
    for a, b in zip(*results):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    for b, s in zip(big, small):
        assert torch.equal(b[far:].view(torch.uint8), s.view(torch.uint8))
        assert not bool(b[:64].view(torch.uint8).any())
