"""The 8-bit cache behind the cache manager, in graphs, on streams, and in the runner."""
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import kv8_util as U
from nanoslg_b200 import ops
from nanoslg_b200.kv_cache import B200PagedKVCache, KVCacheConfig, create_cache_manager
from nanoslg_b200.runner import LlamaRunner, llama_config
from oracle import kv8
from oracle.rope_norm import rope_table

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(autouse=True)
def _clean_status():
    ops.status_word(DEV).zero_()
    yield
    ops.check_device_status(DEV)


def _manager(hq, hkv, d, dt, pages, layers=1, ps=16):
    return B200PagedKVCache(KVCacheConfig(num_layers=layers, num_kv_heads=hkv, num_qo_heads=hq,
                                          head_dim=d, page_size=ps, max_pages=pages, dtype=dt,
                                          device=DEV, kv_dtype="fp8"))


@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("hq,hkv,d,dt,ps", [(32, 8, 128, torch.bfloat16, 16),
                                            (8, 2, 64, torch.float16, 16),
                                            (4, 2, 64, torch.float32, 16),
                                            (6, 3, 96, torch.bfloat16, 5)])
def test_context_steps_are_the_definition(hq, hkv, d, dt, ps, rope):
    """Prompts, decode steps, a shared prefix and a copy on write (its scales copied too):
    pages and attention against the oracle after every forward."""
    mgr = _manager(hq, hkv, d, dt, 80, layers=2, ps=ps)
    oracle = [kv8.Cache(80, hkv, ps, d) for _ in range(2)]
    cos, sin = rope_table(d, 256, 10000.0)
    lens = {"a": 70, "b": 17, "c": 1}
    toks = {s: list(range(100 * i, 100 * i + n)) for i, (s, n) in enumerate(lens.items())}
    for s in lens:
        mgr.allocate_sequence(s, toks[s])
    seed = [0]

    def forward(sids, counts, offsets=None):
        was = {s: list(mgr.seqs[s].block_table) for s in sids}
        ctx = mgr.begin_forward(sids, counts, offsets)
        for s in sids:
            for a, b in zip(was[s], mgr.seqs[s].block_table):
                if a != b:                                  # copied on write
                    for cache in oracle:
                        for name in "kv":
                            cache.v[name][b], cache.s[name][b] = cache.v[name][a], cache.s[name][a]
        width = max(c + o for c, o in zip(counts, offsets or [0] * len(sids)))
        for layer in range(2):
            seed[0] += 10
            q, k, v = (U.rows((len(sids), width, h, d), dt, seed[0] + j, 1.0)
                       for j, h in enumerate((hq, hkv, hkv)))
            args = (q.to(DEV), k.to(DEV), v.to(DEV))
            out = (ctx.attend_rope(layer, *args, cos.to(DEV), sin.to(DEV)) if rope
                   else ctx.attend(layer, *args, hq, hkv)).cpu().view(len(sids), width, hq, d)
            cache = mgr.pool.kv8_layers[layer]
            for b, s in enumerate(sids):
                o, n = (offsets or [0] * len(sids))[b], counts[b]
                st = mgr.seqs[s]
                start = st.num_tokens
                qf, kf = q[b, o:o + n].float().numpy(), k[b, o:o + n].float().numpy()
                if rope:
                    c, t = cos[start:start + n].numpy(), sin[start:start + n].numpy()
                    qf, kf = kv8.rotate(qf, c, t), kv8.rotate(kf, c, t)
                qr = torch.from_numpy(qf).to(dt).double().numpy()
                oracle[layer].append(st.block_table, start, kf, v[b, o:o + n].float().numpy())
                kk, vv = (oracle[layer].read(st.block_table, start + n, name) for name in "kv")
                for i, x in enumerate((kk, vv)):
                    np.testing.assert_array_equal(U.values(cache[i], cache[2 + i], st.block_table, start + n), x)
                want = kv8.attention(qr, kk, vv, 1 / math.sqrt(d))
                vs = U.token_scales(cache[3], st.block_table, start + n, ps)
                bound = U.attention_bound(qr, kk, vv, vs, 1 / math.sqrt(d), want, dt,
                                          U.HALF[dt] if dt != torch.float32 else 0.0)
                assert (np.abs(out[b, o:o + n].double().numpy() - want) <= bound).all(), (s, layer)
        mgr.end_forward(ctx)

    forward(["a", "b", "c"], [70, 17, 1], [0, 53, 69])
    for _ in range(2 * ps + 1 if ps < 16 else 17):          # over a page's end
        forward(["a", "b", "c"], [1, 1, 1])
    forward(["c", "a"], [5, 2], [0, 3])
    # a second sequence with a's prefix, cut back inside a shared page: its next token copies it
    mgr.append_token_ids("a", list(range(900, 960)))
    mgr.release_sequence("a")
    plen = mgr.allocate_sequence("d", toks["a"])
    assert plen > 0 and plen % ps == 0
    mgr.seqs["d"].num_tokens = plen - 2
    page = mgr.seqs["d"].block_table[plen // ps - 1]
    old = [t[page].clone() for t in mgr.pool.kv8_layers[0]]
    forward(["d", "b"], [1, 1])
    assert mgr.seqs["d"].block_table[plen // ps - 1] != page
    for t, o in zip(mgr.pool.kv8_layers[0], old):
        assert torch.equal(t[page].view(torch.uint8), o.view(torch.uint8))
    forward(["d", "b"], [1, 1])


def test_pages_handed_out_again_start_clean():
    """A page whose block went NaN is released and allocated again."""
    mgr = _manager(8, 2, 64, torch.bfloat16, 3)
    for rnd in range(2):
        mgr.allocate_sequence("s", num_tokens=20)
        ctx = mgr.begin_forward(["s"], [20])
        q, k, v = (U.rows((1, 20, h, 64), torch.bfloat16, 5 + h + rnd).to(DEV) for h in (8, 2, 2))
        if rnd == 0:
            k[0, 3, 0, 0] = math.nan
        out = ctx.attend(0, q, k, v, 8, 2)
        assert bool(torch.isfinite(out).all()) == (rnd == 1)
        mgr.end_forward(ctx)
        mgr.release_sequence("s")


@pytest.mark.parametrize("rope", [True, False])
def test_a_decode_step_begins_a_page_handed_out_again(rope):
    """A step planned on the device opens a page whose blocks its last owner left NaN, with rows
    of zeros; the next step adds a small token."""
    hq, hkv, d, dt = 8, 2, 64, torch.bfloat16
    mgr = _manager(hq, hkv, d, dt, 3)
    cos, sin = (t.to(DEV) for t in rope_table(d, 64, 10000.0))

    def forward(n, make):
        ctx = mgr.begin_forward(["s"], [n])
        q, k, v = (make((1, n, h, d), h) for h in (hq, hkv, hkv))
        out = ctx.attend_rope(0, q, k, v, cos, sin) if rope else ctx.attend(0, q, k, v, hq, hkv)
        mgr.end_forward(ctx)
        return out

    def values(shape, seed):
        return U.rows(shape, dt, seed).to(DEV)

    mgr.allocate_sequence("s", num_tokens=20)
    forward(20, lambda shape, seed: torch.full(shape, math.nan, dtype=dt, device=DEV))
    assert bool(torch.isnan(mgr.pool.k_scale[0, 1:]).all())
    mgr.release_sequence("s")
    mgr.allocate_sequence("s", num_tokens=16)
    forward(16, values)
    out = forward(1, lambda shape, seed: torch.zeros(shape, dtype=dt, device=DEV))
    page = mgr.seqs["s"].block_table[1]
    assert bool(torch.isfinite(out).all())
    for t in (mgr.pool.k_scale, mgr.pool.v_scale):
        assert bool((t[0, page] == 0).all())
    out = forward(1, lambda shape, seed: values(shape, seed) / 64)
    assert bool(torch.isfinite(out).all())
    for t in (mgr.pool.k_scale, mgr.pool.v_scale):
        assert bool((t[0, page] > 0).all()) and bool((t[0, page] < 2.0 ** -8).all())


def test_a_sequence_twice_in_a_forward_is_refused():
    mgr = _manager(8, 2, 64, torch.bfloat16, 10)
    mgr.allocate_sequence("s", num_tokens=3)
    with pytest.raises(ValueError, match="only once"):
        mgr.begin_forward(["s", "s"], [1, 1])


def _problem(lens, hq, hkv, d, dt, seed):
    pages = sum(-(-n // 16) for n in lens) + 2
    tables = U.page_lists(lens, 16, pages, seed)
    cache = U.random_cache(pages, hkv, 16, d, DEV, seed)
    q = U.rows((len(lens), hq, d), dt, seed + 1).to(DEV)
    return q, cache, U.csr(tables, lens, 16, DEV)


def test_graphs_and_streams_do_not_share_scratch():
    """Two captured graphs and two eager streams at once, each long enough to split its
    sequences over CTAs: every result is the one computed alone."""
    probs = [_problem([3000 + 700 * i, 900], 32, 8, 128, torch.bfloat16, 40 + i) for i in range(4)]
    alone = [ops.paged_decode_kv8(q, *c, *plan, 0.09) for q, c, plan in probs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in probs]
    graphs, outs = [], []
    for (q, c, plan), st in list(zip(probs, streams))[:2]:
        g = torch.cuda.CUDAGraph()
        out = torch.empty_like(q)
        with torch.cuda.graph(g, stream=streams[0]):       # one capture stream for both
            for _ in range(20):
                ops.paged_decode_kv8(q, *c, *plan, 0.09, out=out)
        graphs.append(g)
        outs.append(out)
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        got = []
        for i, (q, c, plan) in enumerate(probs):
            with torch.cuda.stream(streams[i]):
                if i < 2:
                    graphs[i].replay()
                else:
                    got.append([ops.paged_decode_kv8(q, *c, *plan, 0.09) for _ in range(20)][-1])
        torch.cuda.synchronize()
        for a, b in zip(outs + got, alone):
            assert torch.equal(a, b)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("behind", ["copy", "rmsnorm"])
@pytest.mark.parametrize("rows", [1, 6, 200])
def test_attention_directly_behind_the_work_that_writes_its_list(rows, behind, graph):
    """The page list and the scales are copied into place right before the call, or right before
    a kernel that lets its dependents start early: every route of decode and prefill takes the
    list that was written last, eager and replayed."""
    hq, hkv, d, dt = 8, 2, 128, torch.bfloat16
    lens = [[900, 40, 700, 260], [230, 1000, 201, 800]]
    tables = [U.page_lists([1024] * 4, 16, 300, 7 + i) for i in range(2)]
    cache = U.random_cache(300, hkv, 16, d, DEV, 8)
    lists = []
    for ln, tab in zip(lens, tables):
        ln = [max(n, rows) for n in ln]
        lists.append(U.csr([t[:-(-n // 16)] for t, n in zip(tab, ln)], ln, 16, DEV))
    room = max(x[1].numel() for x in lists)
    now = [torch.zeros_like(lists[0][0]), torch.zeros(room, dtype=torch.int32, device=DEV),
           torch.ones_like(lists[0][2])]
    q = U.rows((4 * rows, hq, d), dt, 11).to(DEV)
    qo = torch.arange(5, dtype=torch.int32, device=DEV) * rows
    x, w = torch.ones(64, 4096, dtype=dt, device=DEV), torch.ones(4096, dtype=dt, device=DEV)

    def call(src):
        for a, b in zip(now, src):
            torch.add(b, 0, out=a[:b.numel()])
        if behind == "rmsnorm":
            ops.rmsnorm_residual(x, w, 1e-5)
        if rows == 1:
            return ops.paged_decode_kv8(q, *cache, *now, 0.09)
        return ops.paged_prefill_kv8(q, qo, rows, *cache, *now, 0.09)

    def alone(src):
        torch.cuda.synchronize()
        if rows == 1:
            return ops.paged_decode_kv8(q, *cache, *src, 0.09)
        return ops.paged_prefill_kv8(q, qo, rows, *cache, *src, 0.09)
    want = [alone(src) for src in lists]
    assert not torch.equal(*want)
    call(lists[0])
    torch.cuda.synchronize()
    if graph:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = [call(lists[i % 2]) for i in range(20)]
        for _ in range(3):
            g.replay()
    else:
        got = [call(lists[i % 2]) for i in range(60)]
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2]), i


def test_append_and_attention_in_a_graph_follow_the_plan():
    """A captured append + decode replayed over plans written into the same buffers."""
    hq, hkv, d, dt = 16, 4, 128, torch.bfloat16
    lens = [40, 17]
    tables = U.page_lists([64, 64], 16, 12, 3)
    caches = [U.random_cache(12, hkv, 16, d, DEV, 6) for _ in range(2)]
    ptr, idx, lpl = U.csr([t[:-(-n // 16)] for t, n in zip(tables, lens)], lens, 16, DEV, spare=3)
    cos, sin = (t.to(DEV) for t in rope_table(d, 128, 10000.0))
    qo = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    rows = [U.rows((2, h, d), dt, 9 + h).to(DEV) for h in (hq, hkv, hkv)]

    def step(cache):
        q = ops.rope_kv8_append(*rows, cos, sin, *cache, qo, 1, ptr, idx, lpl)
        return ops.paged_decode_kv8(q, *cache, ptr, idx, lpl, 0.09)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[1])
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(caches[0])
    for t, u in zip(*caches):
        t.view(torch.uint8).copy_(u.view(torch.uint8))
    for n in range(9):
        lens = [41 + n, 18 + n]
        for t, u in zip((ptr, idx, lpl), U.csr([t[:-(-x // 16)] for t, x in zip(tables, lens)], lens, 16, DEV)):
            t[:u.numel()].copy_(u)
        for i, r in enumerate(rows):
            r.copy_(U.rows(r.shape, dt, 100 * n + i))
        g.replay()
        assert torch.equal(out, step(caches[1]))
        for t, u in zip(*caches):
            assert torch.equal(t.view(torch.uint8), u.view(torch.uint8))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_runner_with_the_8bit_cache(dt):
    """The tiny Llama over the 8-bit cache: graph and eager decode give the same tokens."""
    prompts = [list(range(3, 40)), [5, 6, 7], list(range(90, 118))]
    runs = []
    for graphs in (False, True):
        r = LlamaRunner(llama_config("tiny"), DEV, dtype=dt, max_kv_pages=64, seed=1, kv_cache_dtype="fp8")
        assert r.cache.pool.k.dtype == torch.float8_e4m3fn
        if graphs:
            r.enable_cuda_graphs([3])
        tok = r.prefill(prompts)
        got = [tok]
        for _ in range(20):
            tok = r.decode_step(tok)
            got.append(tok)
        runs.append(torch.stack(got).cpu())
        r.release()
        r.close()
    assert torch.equal(*runs) and bool((runs[0] >= 0).all())


def test_create_cache_manager_takes_the_config_name():
    hf = llama_config("llama-3.1-8b")
    mc = SimpleNamespace(page_size=16, max_kv_pages=8, kv_cache_dtype="fp8")
    mgr = create_cache_manager(hf, None, DEV, torch.bfloat16, mc)
    assert mgr.pool.k.dtype == torch.float8_e4m3fn
    assert mgr.pool.k.shape == (32, 8, 8, 16, 128) and mgr.pool.k_scale.shape == (32, 8, 8)
