"""The 8-bit KV cache at the ends of f32's range, captured calls that cut their
keys, and the kernels and branches that only particular sizes reach.

gpu: each against the model of kv8_model.py in 64 bits, or, replayed from a
     graph, against the eager calls.
"""
import ctypes
import math

import numpy as np
import pytest

from air_amd import capi
from tests.kv8_model import Cache, page_tables
from tests.test_gpu_kv8 import Device, check_weights, rows, same, within

I8, E4M3 = capi.KV8_I8, capi.KV8_E4M3
KINDS = pytest.mark.parametrize("kind", [I8, E4M3], ids=["i8", "e4m3"])
MODES = {None: capi.KV8_WEIGHTS_NONE, "add": capi.KV8_WEIGHTS_ADD, "set": capi.KV8_WEIGHTS_SET}


def filled(kind, kvh, d, lengths, rng, max_pages=None, k_scale=None, page_tokens=16):
    """A cache of one layer whose K of token t is k_scale(sequence, t) times
    an ordinary one, stored by the model's append."""
    pages = max(-(-n // page_tokens) for n in lengths)
    cache = Cache(kind, kvh, d, 1, page_tokens, pages * len(lengths) + 3, max_pages or pages + 2, seed=kind)
    tables = page_tables(rng, lengths, page_tokens, cache.max_pages, cache.pool_pages)
    for i, n in enumerate(lengths):
        x = rows(rng, n, 0, kvh, d, spread=0.5)
        if k_scale is not None:
            x[:, :kvh * d] *= np.array([[k_scale(i, t)] for t in range(n)], dtype=np.float32)
        for a in range(0, n, 2048):
            b = min(n, a + 2048)
            cache.append(x[a:b], 0, list(range(a, b)), np.repeat(tables[i:i + 1], b - a, axis=0), 0)
    return cache, tables


def attend(dev, x, pos, tab, q_heads, max_tokens, runs=None, mode=None):
    """One call checked against the model, output and weights."""
    got = dev.attention(x, pos, tab, 0, q_heads, max_tokens, runs, weights=MODES[mode])
    want, tol, far = dev.cache.attention(x, pos, tab, 0, q_heads, max_tokens, runs, weights=mode)
    print("rows", len(pos), "runs", runs and len(runs), mode, flush=True)
    within(got, want, tol)
    if mode:
        pool = dev.pool()
        check_weights(dev.cache, pool, far)
        dev.cache.pool[...] = pool


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("q_scale,k_scale", [(1.0, 1e-42), (1e-25, 1e-25), (1e-18, 1e-22), (1e-32, 1e-12)])
def test_products_below_f32(torch_cuda, hip_ctx, kind, q_scale, k_scale):
    """q and K whose products lie below f32's range, K of stored scales above
    zero: scores of nothing, so every token weighs the same.  An ordinary block
    lies between such blocks, and one row of ordinary q between such rows."""
    rng = np.random.default_rng(kind + int(-math.log10(q_scale * k_scale)))
    q_heads, kvh, d, n = 14, 2, 128, 600
    cache, tables = filled(kind, kvh, d, [n, 101, 95], rng, k_scale=lambda i, t: 1.0 if t // 16 == 3 else k_scale)
    k_scales = Cache.floats(cache.pool[tables[0, 4], 0, :, 0])[:, 0]
    assert (k_scales > 0).all()
    dev = Device(torch_cuda, hip_ctx, cache)

    def query(m):
        x = rows(rng, m, q_heads, kvh, d)
        x[np.arange(m) != 1] *= np.float32(q_scale)
        return x
    for mode in (None, "set"):
        attend(dev, query(3), [n - 1, 100, 94], tables, q_heads, 110, None, mode)
        attend(dev, query(2), [n - 1, 70], tables[:2], q_heads, n, None, mode)        # cut
        attend(dev, query(40), [60 + t for t in range(40)], np.repeat(tables[:1], 40, axis=0), q_heads, 110, [(0, 40)],
               mode)


@pytest.mark.gpu
@KINDS
def test_queries_up_to_f32s_largest(torch_cuda, hip_ctx, kind):
    """q of 2^126 and more over K as small: ordinary scores."""
    rng = np.random.default_rng(7 + kind)
    q_heads, kvh, d, n = 14, 2, 128, 200
    cache, tables = filled(kind, kvh, d, [n, n], rng, k_scale=lambda i, t: 2.0 ** -126)
    dev = Device(torch_cuda, hip_ctx, cache)
    for m, runs in ((2, None), (40, [(0, 40)])):
        x = rows(rng, m, q_heads, kvh, d)
        x[:, :q_heads * d] = np.clip(x[:, :q_heads * d], -3.9, 3.9) * np.float32(2.0 ** 126)
        assert np.isfinite(x).all() and np.abs(x).max() > 2.0 ** 126
        for mode in (None, "set"):
            tab = np.repeat(tables[:1], m, axis=0) if runs else tables
            attend(dev, x, [n - 1 - r for r in range(m)], tab, q_heads, n, runs, mode)


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [2e6, 3e7, 1e8, 4e8, 1e12, 1e30], ids=lambda s: f"{s:.0e}")
def test_scores_far_past_f32s_whole_numbers(torch_cuda, hip_ctx, kind, d, size):
    """Scores of +-1, 1/2 and 1/4 times `size`.  Tokens of one such score have
    the same codes under the same scale, so whatever a kernel makes of them is
    equal, and the others lie so far below that their part is zero: the tokens
    of the largest score share the weight equally, to the accuracy of p and the
    sums (2^-21 and 6 sqrt(tokens) 2^-24, as the model derives them for scores
    without an error).  Rows of ordinary q between them; cut and uncut keys, a
    run's tiles, weights by every kernel."""
    rng = np.random.default_rng(d + kind + int(math.log10(size)))
    q_heads, kvh, n = 14, 2, 1300
    cache, tables = filled(kind, kvh, d, [n, n, 100], rng)
    sign = np.where(rng.random((kvh, d)) < 0.5, -1.0, 1.0).astype(np.float32)
    part = rng.choice([1.0, 0.5, 0.25], n).astype(np.float32)
    part[::16] = 1.0                                  # every block's scale is that of 1
    part[rng.integers(1, 16)] = 0.25
    x = np.concatenate([(part[:, None, None] * sign).reshape(n, -1),
                        rng.standard_normal((n, kvh * d)).astype(np.float32)], axis=1)
    for i, b in enumerate((n, n, 100)):
        cache.append(x[:b], 0, list(range(b)), np.repeat(tables[i:i + 1], b, axis=0), 0)
    dev = Device(torch_cuda, hip_ctx, cache)
    exact = {"on": False}
    usual = cache.rounding

    def rounding(q, k, tokens):
        ds, rel = usual(q, k, tokens)
        s = np.sort(k @ q / math.sqrt(d))
        if s[-1] - s[0] < 1e5:
            return ds, rel
        exact["on"] = True
        gaps = np.diff(s)
        assert ((gaps == 0) | (gaps > 100 + 2 * ds)).all()
        return 0.0, 2.0 ** -21 + 6 * math.sqrt(tokens) * 2.0 ** -24
    cache.rounding = rounding

    def query(m):
        q = rng.standard_normal((m, kvh, q_heads // kvh, d)).astype(np.float32)
        # Eight bits, so that float64 sums the 128 products without a rounding.
        a = rng.integers(180, 256, q.shape[:3]) * 2.0 ** (math.floor(math.log2(size / math.sqrt(d))) - 8)
        a *= np.where(rng.random(q.shape[:3]) < 0.5, -1, 1)
        far = rng.random(q.shape[:3]) < 0.8
        far[0] = True
        q[far] = (a[..., None] * sign[None, :, None, :]).astype(np.float32)[far]
        return q.reshape(m, -1)
    for mode in (None, "set"):
        attend(dev, query(3), [90, -1, 33], tables, q_heads, 100, None, mode)       # one launch
        attend(dev, query(2), [n - 1, 740], tables[:2], q_heads, n, None, mode)     # cut, joined
        attend(dev, query(24), [n - 3 - 200 * (r % 4) for r in range(24)], np.repeat(tables[:1], 24, axis=0), q_heads, n,
               [(0, 24)], mode)
    assert exact["on"]


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kvh,d", [(28, 4, 128), (14, 2, 64), (40, 1, 64), (8, 8, 128)])
def test_the_largest_call_sizes_the_scratch(torch_cuda, q_heads, kvh, d):
    """After a call of the most rows, runs and tokens with weights, no call of
    fewer grows the scratch: a capture of any of them allocates nothing."""
    torch = torch_cuda
    rng = np.random.default_rng(q_heads + d)
    page_tokens, m, top = 1024, 300, 131072
    stream = torch.cuda.Stream()
    with capi.Context(0, stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        pool = torch.zeros(16, device="cuda:0")
        kv = capi.Kv8Layout(pool.data_ptr(), page_tokens, kvh, d, 1, top // page_tokens, 1, None, 0, I8)
        x = torch.zeros((m, q_heads * d), device="cuda:0")
        out = torch.empty_like(x)
        gone = torch.full((m,), -1, dtype=torch.int32, device="cuda:0")
        tables = torch.full((m, top // page_tokens), -1, dtype=torch.int32, device="cuda:0")

        def call(rows_, runs, tokens, mode):
            starts = None
            if runs:
                cuts = np.sort(rng.integers(0, rows_ + 1, runs - 1))
                starts = torch.tensor([0, *cuts.tolist(), rows_], dtype=torch.int32, device="cuda:0")
            capi.check(capi.lib().air_hip_kv8_attention(
                ctx.handle, ctypes.byref(kv), x.data_ptr(), q_heads * d, rows_, gone.data_ptr(), tables.data_ptr(), 0,
                q_heads, starts.data_ptr() if runs else None, runs, tokens, mode, out.data_ptr()))
            torch.cuda.synchronize()
        call(m, m, top, capi.KV8_WEIGHTS_ADD)
        before = ctx.stats()["workspace_generation"]
        sizes = [(64, 0, 4000), (48, 0, 4000), (32, 0, 4000), (16, 0, 4000), (1, 0, top), (2, 1, top), (m, 1, top),
                 (m, 2, 4000), (60, 2, 320), (33, 33, 70000)]
        for _ in range(150):
            rows_ = int(math.exp(rng.uniform(0, math.log(m + 0.99))))
            runs = int(rng.integers(0, 3)) * int(math.exp(rng.uniform(0, math.log(rows_ + 0.99))))
            sizes.append((rows_, min(runs, m), int(math.exp(rng.uniform(0, math.log(top))))))
        for rows_, runs, tokens in sizes:
            for mode in (capi.KV8_WEIGHTS_NONE, capi.KV8_WEIGHTS_SET):
                call(rows_, runs, tokens, mode)
                assert ctx.stats()["workspace_generation"] == before, (rows_, runs, tokens, mode)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            capi.check(capi.lib().air_hip_kv8_attention(
                ctx.handle, ctypes.byref(kv), x.data_ptr(), q_heads * d, 16, gone.data_ptr(), tables.data_ptr(), 0,
                q_heads, None, 0, 4000, capi.KV8_WEIGHTS_SET, out.data_ptr()))
        out.fill_(1.0)
        g.replay()
        torch.cuda.synchronize()
        assert not out[:16].any() and (out[16:] == 1.0).all()
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kvh,d", [(14, 2, 64), (28, 4, 128)])
def test_captured_calls_that_cut_their_keys(torch_cuda, q_heads, kvh, d):
    """Calls whose keys are cut, each in a graph of its own on one context:
    rows joined in a launch of their own, by a workgroup a vector, and in that
    of the weights; a prompt's tiles with their weights.  Every replay equals
    the eager calls on a copy of the cache, also after an eager call that needed
    a larger scratch, so that the graphs use the one they were captured with."""
    torch = torch_cuda
    rng = np.random.default_rng(151 + d)
    lengths = [5000, 40, 900]
    cache, tables = filled(E4M3, kvh, d, lengths, rng, max_pages=600)
    stream = torch.cuda.Stream()
    with capi.Context(0, stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        dev, ref = Device(torch, ctx, cache), Device(torch, ctx, cache)
        m = 40
        x = dev.up(rows(rng, m, q_heads, kvh, d))
        pos = dev.up([n - 1 for n in lengths], np.int32)
        tab = dev.up(tables, np.int32)
        run_pos = dev.up([4900 + r for r in range(20)] + [850 + r for r in range(20)], np.int32)
        run_tab = dev.up(np.repeat(tables[[0, 2]], 20, axis=0), np.int32)
        starts = dev.up([0, 20, 40], np.int32)
        out = [torch.zeros((m, q_heads * d), device="cuda:0") for _ in range(2)]

        def rows_call(side, y, bound, mode):
            capi.check(side.lib.air_hip_kv8_attention(
                ctx.handle, ctypes.byref(side.kv), x.data_ptr(), x.shape[1], 3, pos.data_ptr(), tab.data_ptr(), 0,
                q_heads, None, 0, bound, mode, y.data_ptr()))

        def runs_call(side, y, bound, mode):
            capi.check(side.lib.air_hip_kv8_attention(
                ctx.handle, ctypes.byref(side.kv), x.data_ptr(), x.shape[1], m, run_pos.data_ptr(), run_tab.data_ptr(),
                0, q_heads, starts.data_ptr(), 2, bound, mode, y.data_ptr()))
        kinds = [(rows_call, 1500, capi.KV8_WEIGHTS_NONE), (rows_call, 1500, capi.KV8_WEIGHTS_ADD),
                 (rows_call, 9600, capi.KV8_WEIGHTS_NONE), (rows_call, 9600, capi.KV8_WEIGHTS_ADD),
                 (runs_call, 5000, capi.KV8_WEIGHTS_SET), (runs_call, 5000, capi.KV8_WEIGHTS_ADD)]
        for call, bound, mode in kinds:
            for side in (dev, ref):
                call(side, out[0], bound, mode)       # sizes the scratch
        torch.cuda.synchronize()
        before = ctx.stats()["workspace_generation"]
        graphs = []
        for call, bound, mode in kinds:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                call(dev, out[0], bound, mode)
            graphs.append(g)
        assert ctx.stats()["workspace_generation"] == before

        def grow():
            many = 1000
            wide = torch.zeros((many, q_heads * d), device="cuda:0")
            gone = torch.full((many,), -1, dtype=torch.int32, device="cuda:0")
            none = torch.full((many, cache.max_pages), -1, dtype=torch.int32, device="cuda:0")
            ends = dev.up([0, many], np.int32)
            capi.check(dev.lib.air_hip_kv8_attention(
                ctx.handle, ctypes.byref(dev.kv), wide.data_ptr(), q_heads * d, many, gone.data_ptr(), none.data_ptr(),
                0, q_heads, ends.data_ptr(), 1, 5000, capi.KV8_WEIGHTS_ADD, wide.data_ptr()))
            torch.cuda.synchronize()
            assert ctx.stats()["workspace_generation"] > before
        for turn in range(3):
            if turn == 1:
                grow()
            for g, (call, bound, mode) in zip(graphs, kinds):
                x.copy_(dev.up(rows(rng, m, q_heads, kvh, d)))
                for y in out:
                    y.zero_()
                torch.cuda.synchronize()
                g.replay()
                call(ref, out[1], bound, mode)
                torch.cuda.synchronize()
                assert out[0].any() and torch.equal(out[0], out[1]), (turn, call.__name__, bound, mode)
                assert same(dev.pool(), ref.pool()), (turn, call.__name__, bound, mode)
    torch.cuda.synchronize()


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("kvh,d,page_tokens", [(4, 128, 16), (3, 64, 32)])
def test_read_of_the_weights_alone(torch_cuda, hip_ctx, kind, kvh, d, page_tokens):
    """No k and no v asked for: from the start and from inside a block, past
    max_tokens, without a page, of no tokens; the rest of the buffer stays."""
    torch = torch_cuda
    rng = np.random.default_rng(17 + kind)
    lengths = [150, 1, 77, 33]
    cache = Cache(kind, kvh, d, 3, page_tokens, 40, 12, seed=3)
    tables = page_tables(rng, lengths, page_tokens, 12, 40)
    tables[2, 1] = -1
    dev = Device(torch, hip_ctx, cache)
    for starts, counts, layer, layers, top in ((None, lengths, 1, 2, 150), ([5, 0, 30, 33], [90, 1, 40, 0], 0, 3, 64),
                                               ([-1, 0, 16, 31], [9, 0, 48, 2], 2, 1, 48)):
        w = torch.full((layers, 4, top, kvh), 7.0, device="cuda:0")
        s = dev.up(starts, np.int32) if starts else None
        n, t = dev.up(counts, np.int32), dev.up(tables, np.int32)
        capi.check(dev.lib.air_hip_kv8_read(hip_ctx.handle, ctypes.byref(dev.kv), 4, s.data_ptr() if starts else None,
                                            n.data_ptr(), t.data_ptr(), layer, layers, top, None, None, w.data_ptr()))
        torch.cuda.synchronize()
        counts = [0 if starts and a < 0 else c for a, c in zip(starts or lengths, counts)]
        want = cache.read(starts, counts, tables, layer, layers, top, 7.0)[2]
        assert np.array_equal(w.cpu().numpy(), want)


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("kvh,d", [(4, 128), (2, 64)])
def test_append_and_read_of_unaligned_rows(torch_cuda, hip_ctx, kind, kvh, d):
    """Rows that begin 4 bytes past an alignment, of odd strides, with k behind
    a q of odd width; values read to such buffers."""
    torch = torch_cuda
    rng = np.random.default_rng(27 + kind)
    n, width = 53, 2 * kvh * d
    for offset, pad, q_width in ((1, 0, 4), (0, 1, 4), (0, 0, 3), (3, 5, 7)):
        cache = Cache(kind, kvh, d, 1, 16, 6, 5, seed=9)
        table = page_tables(rng, [n], 16, 5, 6)
        dev = Device(torch, hip_ctx, cache)
        stride = q_width + width + pad
        x = rng.standard_normal((n, stride)).astype(np.float32)
        buf = torch.zeros(offset + n * stride, device="cuda:0")
        buf[offset:] = dev.up(x).reshape(-1)
        pos, tab = dev.up(list(range(n)), np.int32), dev.up(np.repeat(table, n, axis=0), np.int32)
        capi.check(dev.lib.air_hip_kv8_append(hip_ctx.handle, ctypes.byref(dev.kv), buf.data_ptr() + 4 * offset, stride,
                                              q_width, n, pos.data_ptr(), tab.data_ptr(), 0))
        cache.append(x, q_width, list(range(n)), np.repeat(table, n, axis=0), 0)
        assert same(dev.pool(), cache.pool), (offset, pad, q_width)
        size = (n + 2) * kvh * d
        for at_k, at_v in ((1, 0), (0, 3), (2, 1)):
            k, v = (torch.full((at + size + 1,), 7.0, device="cuda:0") for at in (at_k, at_v))
            count = dev.up([n], np.int32)
            capi.check(dev.lib.air_hip_kv8_read(hip_ctx.handle, ctypes.byref(dev.kv), 1, None, count.data_ptr(),
                                                tab.data_ptr(), 0, 1, n + 2, k.data_ptr() + 4 * at_k,
                                                v.data_ptr() + 4 * at_v, None))
            torch.cuda.synchronize()
            want_k, want_v, _ = cache.read(None, [n], table, 0, 1, n + 2, 7.0)
            for got, want, at in ((k, want_k, at_k), (v, want_v, at_v)):
                got = got.cpu().numpy()
                assert np.array_equal(got[at:at + size], want.reshape(-1))
                assert (got[:at] == 7.0).all() and got[-1] == 7.0


def runs_of(lengths, rows_of, tables, empty_every):
    """Rows at the end of each sequence, as runs with empty ones between."""
    pos, tab, runs = [], [], []
    for i, (n, b) in enumerate(zip(lengths, rows_of)):
        runs.append((len(pos), len(pos) + b))
        if i % empty_every == 0:
            runs.append((len(pos) + b, len(pos) + b))
        pos += range(n - b, n)
        tab += [tables[i]] * b
    return pos, np.array(tab), runs


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("q_heads,kvh,d", [(14, 2, 64), (6, 2, 128)])
def test_many_ragged_runs_in_tiles_of_rows(torch_cuda, hip_ctx, kind, q_heads, kvh, d):
    """More runs than a wave looks up at a time, of one to nineteen rows, in
    tiles of four and of ten rows; empty runs among them and at both ends."""
    rng = np.random.default_rng(161 + kind + d)
    rows_of = [int(b) for b in rng.integers(1, 20, 75)]
    lengths = [int(a) + b for a, b in zip(rng.integers(0, 40, 75), rows_of)]
    cache, tables = filled(kind, kvh, d, lengths, rng, max_pages=30)
    pos, tab, runs = runs_of(lengths, rows_of, tables, 8)
    runs = [(0, 0)] + runs + [(len(pos), len(pos))] * 2
    dev = Device(torch_cuda, hip_ctx, cache)
    for mode in (None, "set", "add"):
        attend(dev, rows(rng, len(pos), q_heads, kvh, d), pos, tab, q_heads, 480, runs, mode)


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("d", [64, 128])
def test_runs_tiles_with_a_wave_a_chunk_of_weights(torch_cuda, hip_ctx, kind, d):
    """Runs of many vectors over keys that may be long: tiles, some of them
    cut, whose weights a wave a chunk gathers."""
    rng = np.random.default_rng(171 + kind + d)
    q_heads, kvh, runs_n, b = 14, 2, 24, 12
    lengths = [1450, 1300] + [int(n) for n in rng.integers(b, 60, runs_n - 2)]
    cache, tables = filled(kind, kvh, d, lengths, rng, max_pages=208)
    pos, tab, runs = runs_of(lengths, [b] * runs_n, tables, 100)
    dev = Device(torch_cuda, hip_ctx, cache)
    for mode in ("set", "add"):
        attend(dev, rows(rng, len(pos), q_heads, kvh, d), pos, tab, q_heads, 208 * 16, runs, mode)


@pytest.mark.gpu
@KINDS
def test_rows_for_most_of_the_card_are_not_cut(torch_cuda, hip_ctx, kind):
    """Forty rows of four KV heads under a bound far above most of them: a
    workgroup a (row, KV head) takes all chunks, without and with weights."""
    rng = np.random.default_rng(181 + kind)
    q_heads, kvh, d = 8, 4, 128
    lengths = [2700] + [int(n) for n in rng.integers(1, 90, 39)]
    cache, tables = filled(kind, kvh, d, lengths, rng)
    dev = Device(torch_cuda, hip_ctx, cache)
    for mode in (None, "add", "set"):
        attend(dev, rows(rng, 40, q_heads, kvh, d), [n - 1 for n in lengths], tables, q_heads, 2720, None, mode)
