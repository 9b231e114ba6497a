"""The 8-bit KV cache: append, read, attention with its weights, eviction.

cpu: page sizes, null arguments, and the model's own rounding.
gpu: the stored bytes of append and eviction equal the model's (kv8_model.py)
     bit for bit; attention and the weights lie within the bounds that its
     `rounding` derives of a float64 attention over the same codes; a serving
     run of all of them, eager and captured.
"""
import ctypes

import numpy as np
import pytest

from air_amd import capi
from tests import kv8_model
from tests.kv8_model import Cache, page_tables

I8, E4M3 = capi.KV8_I8, capi.KV8_E4M3
KINDS = pytest.mark.parametrize("kind", [I8, E4M3], ids=["i8", "e4m3"])


# ---- cpu --------------------------------------------------------------------

def test_page_bytes():
    lay = capi.Kv8Layout(None, 48, 4, 128, 3, 7, 9, None, 0, I8)
    assert capi.kv8_page_bytes(lay) == 3 * 4 * 3 * (128 + 32 * 128)
    lay.head_dim = 64
    assert capi.kv8_page_bytes(lay) == 3 * 4 * 3 * (128 + 32 * 64)
    for field, bad in [("page_tokens", 24), ("page_tokens", 0), ("head_dim", 96), ("kv_heads", 0), ("layers", 0),
                       ("type", 0), ("type", 3), ("max_pages", 0), ("pool_pages", 0), ("max_pages", 2 ** 31),
                       ("pool_pages", 2 ** 31), ("page_tokens", 65552), ("layers", 65535)]:
        broken = capi.Kv8Layout(None, 48, 12, 64, 3, 7, 9, None, 0, I8)
        setattr(broken, field, bad)
        assert capi.kv8_page_bytes(broken) == 0, (field, bad)
    assert capi.lib().air_hip_kv8_page_bytes(None) == 0


def test_null_arguments():
    lib = capi.lib()
    lay = ctypes.byref(capi.Kv8Layout(16, 16, 4, 128, 1, 1, 1, None, 0, I8))
    assert lib.air_hip_kv8_append(None, lay, 16, 2048, 1024, 1, 16, 16, 0) == 1
    assert lib.air_hip_kv8_read(None, lay, 1, None, 16, 16, 0, 1, 16, 16, 16, 16) == 1
    assert lib.air_hip_kv8_attention(None, lay, 16, 2048, 1, 16, 16, 0, 8, None, 0, 16, 0, 16) == 1
    assert lib.air_hip_kv8_evict(None, lay, 1, 16, 16, 16, 0, 1, 0, 0, 8, 16, 16) == 1
    assert b"null" in lib.air_hip_last_error()


def test_model_rounds_like_torch():
    """The model's e4m3 codes are torch's, ties and both ends included."""
    torch = pytest.importorskip("torch")
    rng = np.random.default_rng(1)
    mags = kv8_model.E4M3[:127]
    mids = (mags[1:] + mags[:-1]) / 2
    x = np.concatenate([mags, mids, np.nextafter(mids.astype(np.float32), np.float32(0)), [448.0],
                        rng.uniform(0, 448, 4096)]).astype(np.float32)
    x = np.concatenate([x, -x])
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(kv8_model.encode(x, E4M3), want)


# ---- gpu --------------------------------------------------------------------

class Device:
    """A model cache and its copy on the GPU, called through the C ABI."""

    def __init__(self, torch, ctx, cache, chunk_shift=None):
        self.torch, self.ctx, self.cache, self.lib = torch, ctx, cache, capi.lib()
        self.dev = torch.device("cuda:0")
        if chunk_shift is None:
            self.parts = [torch.from_numpy(cache.pool.copy()).to(self.dev)]
            self.kv = cache.layout(self.parts[0].data_ptr())
        else:
            per = 1 << chunk_shift
            self.parts = [torch.from_numpy(cache.pool[i:i + per].copy()).to(self.dev)
                          for i in range(0, cache.pool_pages, per)]
            self.bases = torch.tensor([p.data_ptr() for p in self.parts], dtype=torch.int64, device=self.dev)
            self.kv = cache.layout(None, self.bases.data_ptr(), chunk_shift)

    def up(self, a, dtype=None):
        return self.torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype=dtype))).to(self.dev)

    def pool(self):
        self.torch.cuda.synchronize()
        return np.concatenate([p.cpu().numpy() for p in self.parts])

    def append(self, qkv, q_width, positions, tables, layer):
        x, p, t = self.up(qkv), self.up(positions, np.int32), self.up(tables, np.int32)
        capi.check(self.lib.air_hip_kv8_append(self.ctx.handle, ctypes.byref(self.kv), x.data_ptr(), x.shape[1],
                                               q_width, len(positions), p.data_ptr(), t.data_ptr(), layer))
        self.torch.cuda.synchronize()

    def attention(self, qkv, positions, tables, layer, q_heads, max_tokens, runs=None, weights=0):
        x, p, t = self.up(qkv), self.up(positions, np.int32), self.up(tables, np.int32)
        out = self.torch.full((len(positions), q_heads * self.cache.d), float("nan"), device=self.dev)
        starts = None if runs is None else self.up([b for b, _ in runs] + [runs[-1][1]], np.int32)
        capi.check(self.lib.air_hip_kv8_attention(
            self.ctx.handle, ctypes.byref(self.kv), x.data_ptr(), x.shape[1], len(positions), p.data_ptr(),
            t.data_ptr(), layer, q_heads, starts.data_ptr() if runs else None, len(runs) if runs else 0, max_tokens,
            weights, out.data_ptr()))
        self.torch.cuda.synchronize()
        return out.cpu().numpy()

    def evict(self, lengths, tables, new_tables, layer, layers, keep_first, keep_last, budget, max_tokens):
        n, t = self.up(lengths, np.int32), self.up(tables, np.int32)
        new = t if new_tables is tables else self.up(new_tables, np.int32)
        kept = self.torch.full((len(lengths), layers, self.cache.kvh, budget), -7, dtype=self.torch.int32,
                               device=self.dev)
        capi.check(self.lib.air_hip_kv8_evict(self.ctx.handle, ctypes.byref(self.kv), len(lengths), n.data_ptr(),
                                              t.data_ptr(), new.data_ptr(), layer, layers, keep_first, keep_last,
                                              budget, max_tokens, kept.data_ptr()))
        self.torch.cuda.synchronize()
        return kept.cpu().numpy()

    def read(self, starts, lengths, tables, layer, layers, max_tokens, fill):
        c = self.cache
        n, t = self.up(lengths, np.int32), self.up(tables, np.int32)
        s = self.up(starts, np.int32) if starts else None
        shape = (layers, len(lengths), max_tokens, c.kvh * c.d)
        k = self.torch.full(shape, fill, device=self.dev)
        v = self.torch.full(shape, fill, device=self.dev)
        w = self.torch.full(shape[:3] + (c.kvh,), fill, device=self.dev)
        capi.check(self.lib.air_hip_kv8_read(self.ctx.handle, ctypes.byref(self.kv), len(lengths),
                                             s.data_ptr() if starts else None, n.data_ptr(), t.data_ptr(), layer,
                                             layers, max_tokens, k.data_ptr(), v.data_ptr(), w.data_ptr()))
        self.torch.cuda.synchronize()
        return k.cpu().numpy(), v.cpu().numpy(), w.cpu().numpy()


def same(a, b):
    """Bit equality, NaN payloads aside (both are the cache's only NaN scale)."""
    a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
    if a.dtype == np.uint8:
        fa, fb = a[..., :128].copy().view(np.float32), b[..., :128].copy().view(np.float32)
        return np.array_equal(fa, fb, equal_nan=True) and np.array_equal(a[..., 128:], b[..., 128:])
    return np.array_equal(a, b, equal_nan=True)


def rows(rng, m, q_heads, kvh, d, pad=0, spread=1.0):
    """q|k|v rows with values of several magnitudes."""
    width = q_heads * d + 2 * kvh * d
    x = rng.standard_normal((m, width + pad)).astype(np.float32)
    x[:, q_heads * d:width] *= np.exp(spread * rng.standard_normal((m, 1))).astype(np.float32)
    return x


def within(got, want, tol):
    bad = ~(np.abs(got.astype(np.float64) - want) <= tol)
    assert not bad.any(), (int(bad.sum()), float(np.max(np.abs(got - want) / tol)), np.argwhere(bad)[:3].tolist())


def check_weights(cache, pool, far):
    got = Cache.__new__(Cache)
    got.__dict__.update(cache.__dict__)
    got.pool = pool
    for table, layer, g, t, tol in far:
        a, b = cache.slot(table, layer, g, t), got.slot(table, layer, g, t)
        x, y = float(Cache.floats(a[0])[16 + a[1]]), float(Cache.floats(b[0])[16 + b[1]])
        assert abs(x - y) <= tol, (layer, g, t, x, y, tol)


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("kvh,d,page_tokens", [(4, 128, 16), (2, 64, 48)])
def test_append_stores_the_models_bytes(torch_cuda, hip_ctx, kind, kvh, d, page_tokens):
    """Successive calls: fresh blocks, blocks that go on (with and without a
    larger scale), rows out of order, one slot twice, a padded stride, rows
    without a position or a page, zeros, an infinity, a NaN, a new beginning."""
    rng = np.random.default_rng(d + kind)
    lengths = [70, 5, 33]
    cache = Cache(kind, kvh, d, 2, page_tokens, 20, 6, seed=kind)
    tables = page_tables(rng, [96, 96, 96], page_tokens, 6, 20)
    dev = Device(torch_cuda, hip_ctx, cache)
    q_heads, qw = 2 * kvh, 2 * kvh * d

    def step(named, change=None, pad=0, layer=1):
        order = rng.permutation(len(named))
        named = [named[i] for i in order]
        x = rows(rng, len(named), q_heads, kvh, d, pad)
        if change:
            change(x, named)
        pos = [p for _, p in named]
        tab = tables[[s for s, _ in named]]
        dev.append(x, qw, pos, tab, layer)
        cache.append(x, qw, pos, tab, layer)
        print("rows", len(named), flush=True)
        assert same(dev.pool(), cache.pool)

    step([(s, p) for s, n in enumerate(lengths) for p in range(n)])
    step([(0, 70), (1, 5), (2, 33)], pad=8)
    step([(0, 71), (1, 6), (2, 34), (0, 71), (0, 71), (1, -1), (2, 95), (2, 6 * page_tokens)])
    step([(0, 72 + i) for i in range(30)] + [(1, 7)], lambda x, named: x.__imul__(np.float32(40.0)))
    step([(1, 16 + i) for i in range(16)], lambda x, named: x[:, qw:].fill(0.0))
    step([(2, 35), (2, 36)], lambda x, named: x[:, qw:].fill(0.0))

    def broken(x, named):
        at = {p: i for i, (_, p) in enumerate(named)}
        x[at[37], qw + 3] = np.inf                     # K of head 0
        x[at[38], qw + kvh * d + d] = np.nan           # V of head 1
    step([(2, 37), (2, 38)], broken)
    step([(2, 39)])                                    # goes on in a poisoned block
    step([(2, 32), (2, 33)])                           # begins it anew
    step([(0, 0)], lambda x, named: x.__imul__(np.float32(1e-42)), layer=0)   # scales below f32's normal range


@pytest.mark.gpu
@KINDS
def test_append_of_many_rows_runs_in_slices(torch_cuda, hip_ctx, kind):
    """2048 rows are one call, more are successive ones; a block that lies
    across the seam is quantised in two steps."""
    rng = np.random.default_rng(5)
    n, start, kvh, d = 2100, 9, 1, 64
    cache = Cache(kind, kvh, d, 1, 16, 140, 140)
    table = page_tables(rng, [n + start], 16, 140, 140)
    dev = Device(torch_cuda, hip_ctx, cache, chunk_shift=2)
    x = rows(rng, n, 1, kvh, d)
    pos = list(range(start, start + n))
    tab = np.repeat(table, n, axis=0)
    dev.append(x, d, pos, tab, 0)
    for a in range(0, n, 2048):
        cache.append(x[a:a + 2048], d, pos[a:a + 2048], tab[a:a + 2048], 0)
    assert same(dev.pool(), cache.pool)


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("kvh,d,page_tokens", [(4, 128, 16), (3, 64, 32)])
def test_read_leaves_the_rest(torch_cuda, hip_ctx, kind, kvh, d, page_tokens):
    rng = np.random.default_rng(d)
    cache = Cache(kind, kvh, d, 3, page_tokens, 12, 5, seed=2)
    if kind == E4M3:
        codes = cache.pool[..., 128:]
        codes[(codes & 127) == 127] = 0               # stored codes are never NaN
    tables = page_tables(rng, [5 * page_tokens, 70, 1], page_tokens, 5, 12)
    tables[0, 1] = -1
    dev = Device(torch_cuda, hip_ctx, cache)
    top = 5 * page_tokens
    for starts, lengths, layer, layers, most in [(None, [top, 70, 1], 0, 3, top), ([17, 3, 0], [20, 0, 1], 1, 2, 40),
                                                 ([15, 16, 0], [40, 2, -3], 2, 1, 33)]:
        got = dev.read(starts, lengths, tables, layer, layers, most, 7.5)
        want = cache.read(starts, lengths, tables, layer, layers, most, 7.5)
        for a, b in zip(got, want):
            assert same(a, b), (starts, lengths)


def _filled(kind, kvh, d, page_tokens, lengths, rng, layers=2, layer=1, spread=0.7, max_pages=None):
    """A cache whose sequences were appended, block by block."""
    max_pages = max_pages or max(1, max(-(-n // page_tokens) for n in lengths))
    pool = sum(-(-n // page_tokens) for n in lengths) + 2
    cache = Cache(kind, kvh, d, layers, page_tokens, pool, max_pages, seed=3)
    tables = page_tables(rng, lengths, page_tokens, max_pages, pool)
    for i, n in enumerate(lengths):
        for a in range(0, n, 2048):
            b = min(n, a + 2048)
            x = rows(rng, b - a, 0, kvh, d, spread=spread)
            cache.append(x, 0, list(range(a, b)), np.repeat(tables[i:i + 1], b - a, axis=0), layer)
    return cache, tables


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("q_heads,kvh,d,page_tokens,lengths", [
    (28, 4, 128, 16, [1, 15, 16, 17, 63, 64, 65, 700]),
    (14, 2, 64, 48, [1, 49, 300, 511, 512, 513]),
    (5, 5, 128, 32, [33, 129]),                       # one q head a KV head
    (40, 1, 64, 16, [200, 3]),                        # forty: three parts
    (16, 1, 128, 64, [1030]),
])
def test_decode_attention(torch_cuda, hip_ctx, kind, q_heads, kvh, d, page_tokens, lengths):
    """One row a sequence, a padding row among them, with and without a bound
    far above the lengths; weights added and set."""
    rng = np.random.default_rng(q_heads * d + kind)
    cache, tables = _filled(kind, kvh, d, page_tokens, lengths, rng)
    dev = Device(torch_cuda, hip_ctx, cache)
    wide = np.full((len(lengths) + 1, cache.max_pages), -1, dtype=np.int32)
    wide[1:] = tables
    pos = [-1] + [n - 1 for n in lengths]
    for max_tokens in sorted({max(lengths), cache.max_pages * page_tokens, max(1, max(lengths) - 3)}):
        x = rows(rng, len(pos), q_heads, kvh, d, pad=4)
        got = dev.attention(x, pos, wide, 1, q_heads, max_tokens)
        want, tol, _ = cache.attention(x, pos, wide, 1, q_heads, max_tokens)
        assert (got[0] == 0).all()
        within(got, want, tol)
    before = dev.pool()
    assert same(before, cache.pool)                   # a plain attention stores nothing
    for mode, name in ((capi.KV8_WEIGHTS_ADD, "add"), (capi.KV8_WEIGHTS_SET, "set"), (capi.KV8_WEIGHTS_ADD, "add")):
        x = rows(rng, len(pos), q_heads, kvh, d)
        got = dev.attention(x, pos, wide, 1, q_heads, max(lengths), weights=mode)
        want, tol, far = cache.attention(x, pos, wide, 1, q_heads, max(lengths), weights=name)
        within(got, want, tol)
        pool = dev.pool()
        check_weights(cache, pool, far)
        assert np.array_equal(pool[..., 128:], cache.pool[..., 128:])
        cache.pool[...] = pool                        # go on from the device's weights
    # Only the tokens attended to changed: what lies behind them keeps its weight.
    for i, n in enumerate(lengths):
        for t in range(n, min(-(-n // 16) * 16, cache.max_pages * page_tokens)):
            at = cache.slot(tables[i], 1, 0, t)
            ref = before[tables[i][t // page_tokens], 1, 0, t % page_tokens // 16]
            assert Cache.floats(at[0])[16 + t % 16] == ref.view(np.float32)[16 + t % 16]


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("q_heads,kvh,d,page_tokens,seqs", [
    # (tokens before the run, rows of the run) of each sequence
    (28, 4, 128, 16, [(0, 37), (50, 1), (3, 64), (200, 5)]),
    (6, 6, 64, 16, [(0, 1), (0, 130), (63, 66)]),
    (14, 2, 64, 32, [(0, 2), (31, 33), (500, 17)]),
    (33, 1, 128, 48, [(10, 9)]),
])
def test_prompt_attention(torch_cuda, hip_ctx, kind, q_heads, kvh, d, page_tokens, seqs):
    """Runs of rows with causal attention, an empty run among them; weights
    set by a run are the sums over its rows."""
    rng = np.random.default_rng(q_heads + d + kind)
    lengths = [a + b for a, b in seqs]
    cache, tables = _filled(kind, kvh, d, page_tokens, lengths, rng)
    dev = Device(torch_cuda, hip_ctx, cache)
    pos, tab, runs = [], [], []
    for i, (a, b) in enumerate(seqs):
        runs.append((len(pos), len(pos) + b))
        if i == 0:
            runs.append((len(pos) + b, len(pos) + b))
        pos += range(a, a + b)
        tab += [tables[i]] * b
    tab = np.array(tab)
    x = rows(rng, len(pos), q_heads, kvh, d)
    got = dev.attention(x, pos, tab, 1, q_heads, max(lengths), runs)
    want, tol, _ = cache.attention(x, pos, tab, 1, q_heads, max(lengths), runs)
    within(got, want, tol)
    got = dev.attention(x, pos, tab, 1, q_heads, max(lengths), runs, weights=capi.KV8_WEIGHTS_SET)
    want, tol, far = cache.attention(x, pos, tab, 1, q_heads, max(lengths), runs, weights="set")
    within(got, want, tol)
    check_weights(cache, dev.pool(), far)
    again = dev.attention(x, pos, tab, 1, q_heads, max(lengths), runs, weights=capi.KV8_WEIGHTS_SET)
    assert np.array_equal(got, again)                 # and every bit of it again


@pytest.mark.gpu
@KINDS
def test_attention_where_it_can_go_wrong(torch_cuda, hip_ctx, kind):
    """Pages missing inside a sequence, blocks of zeros, of values 2^40 apart,
    a query of zeros, scores far apart, stale codes (NaN ones too) behind the
    last token, a poisoned block seen by one row and not by another."""
    rng = np.random.default_rng(11 + kind)
    q_heads, kvh, d, page_tokens = 8, 2, 128, 16
    lengths = [150, 40, 90, 20, 100]
    cache, tables = _filled(kind, kvh, d, page_tokens, lengths, rng)
    tables[0, 2] = -1
    tables[0, 5] = cache.pool_pages                   # out of range: no page

    def rewrite(i, a, b, factor_k, factor_v):
        x = rows(rng, b - a, 0, kvh, d, spread=0.0)
        x[:, :kvh * d] *= np.float32(factor_k)
        x[:, kvh * d:] *= np.float32(factor_v)
        cache.append(x, 0, list(range(a, b)), np.repeat(tables[i:i + 1], b - a, axis=0), 1)
    rewrite(1, 0, 16, 0.0, 0.0)                       # sequence 1: zeros, then ordinary, then large V
    rewrite(1, 32, 40, 1.0, 2.0 ** 40)
    for a in range(0, 90, 16):                        # sequence 2: V from 2^-40 up
        rewrite(2, a, min(a + 16, 90), 0.2, 2.0 ** (a / 2 - 40))
    rewrite(3, 0, 16, 1.0, 0.0)                       # sequence 3: V of zeros and little else
    rewrite(3, 16, 20, 1.0, 1e-30)
    bad = rows(rng, 1, 0, kvh, d)
    bad[0, 5] = np.nan
    bad[0, 2 * kvh * d - 1] = np.inf                  # V of the last KV head
    cache.append(bad, 0, [99], tables[4:5], 1)        # sequence 4: its last block is poisoned
    dev = Device(torch_cuda, hip_ctx, cache)
    named = [(0, 149), (1, 39), (1, 15), (1, 31), (2, 89), (3, 19), (3, 15), (4, 95)]
    pos, tab = [p for _, p in named], tables[[s for s, _ in named]]
    x = rows(rng, len(named), q_heads, kvh, d)
    x[0, :d] = 0.0
    x[1, d:2 * d] *= np.float32(60.0)                 # scores hundreds apart
    x[4, :d] *= np.float32(1e-30)
    got = dev.attention(x, pos, tab, 1, q_heads, 160 - 10)
    want, tol, _ = cache.attention(x, pos, tab, 1, q_heads, 150)
    within(got, want, tol)
    poisoned = dev.attention(x[:2], [99, 39], tables[[4, 1]], 1, q_heads, 150)
    assert np.isnan(poisoned[0, :q_heads // kvh * d]).all()      # K of KV head 0
    assert np.isnan(poisoned[0, -d:]).all() and np.isnan(poisoned[0]).all()   # V of KV head 1
    assert np.isfinite(poisoned[1]).all()
    broken = x[:2].copy()
    broken[0, 3] = np.nan
    got = dev.attention(broken, [149, 39], tables[[0, 1]], 1, q_heads, 150)
    assert np.isnan(got[0, :d]).all() and np.isfinite(got[0, d:]).all() and np.isfinite(got[1]).all()


@pytest.mark.gpu
@KINDS
def test_attention_over_a_long_cache(torch_cuda, hip_ctx, kind):
    """A cache whose pages lie past 4 GiB of the pool, 5000 tokens, and the
    same through chunks."""
    torch = torch_cuda
    rng = np.random.default_rng(21)
    q_heads, kvh, d, page_tokens, n = 4, 2, 128, 64, 5000
    cache, tables = _filled(kind, kvh, d, page_tokens, [n], rng, layers=1, layer=0)
    page = cache.pool[0].nbytes
    far = (5 << 30) // page                           # pages before ours
    pool = torch.empty((far + cache.pool_pages) * page, dtype=torch.uint8, device="cuda:0")
    pool[far * page:] = torch.from_numpy(cache.pool.reshape(-1)).to("cuda:0")
    dev = Device(torch, hip_ctx, cache)
    x = rows(rng, 2, q_heads, kvh, d)
    pos, tab = [n - 1, 2500], np.repeat(tables, 2, axis=0)
    want, tol, _ = cache.attention(x, pos, tab, 0, q_heads, n)
    within(dev.attention(x, pos, tab, 0, q_heads, n), want, tol)
    dev.kv = capi.Kv8Layout(pool.data_ptr(), page_tokens, kvh, d, 1, cache.max_pages, far + cache.pool_pages, None, 0,
                            kind)
    got = dev.attention(x, pos, tab + far, 0, q_heads, n)
    within(got, want, tol)
    chunked = Cache(kind, kvh, d, 1, page_tokens, -(-cache.pool_pages // 4) * 4, cache.max_pages)
    chunked.pool[:cache.pool_pages] = cache.pool
    other = Device(torch, hip_ctx, chunked, chunk_shift=2)
    assert np.array_equal(other.attention(x, pos, tab, 0, q_heads, n), got)
    other.bases[2] = 0                                # a chunk that is not there holds no tokens
    gone = tab.copy()
    gone[(tab >= 8) & (tab < 12)] = -1
    want, tol, _ = cache.attention(x, pos, gone, 0, q_heads, n)
    within(other.attention(x, pos, tab, 0, q_heads, n), want, tol)


@pytest.mark.gpu
@KINDS
def test_attention_errors_are_those_of_f32(torch_cuda, hip_ctx, kind):
    """Over 448 vectors and 3500 tokens the errors against float64 are, in the
    root mean square, at most 16 half steps of f32 (2^-24 each): a score of up
    to 30 is right to about 2^-24 of itself, which e^s turns into a relative
    error of some half steps of p, and the sums add one or two more.  A single
    weight in a thousand held to one f16 (2^-12) would be above it."""
    torch = torch_cuda
    gen = torch.Generator(device="cuda:0")
    gen.manual_seed(61 + kind)
    q_heads, kvh, d, n, m = 28, 4, 128, 3500, 16
    cache = Cache(kind, kvh, d, 1, 16, 224, 224)
    dev = Device(torch, hip_ctx, cache)
    table = torch.randperm(224, device="cuda:0", generator=gen).to(torch.int32).repeat(2048, 1)
    width = 2 * kvh * d
    for a in range(0, n, 2048):
        b = min(n, a + 2048)
        x = torch.randn((b - a, width), device="cuda:0", generator=gen)
        pos = torch.arange(a, b, dtype=torch.int32, device="cuda:0")
        capi.check(dev.lib.air_hip_kv8_append(hip_ctx.handle, ctypes.byref(dev.kv), x.data_ptr(), width, 0, b - a,
                                              pos.data_ptr(), table.data_ptr(), 0))
    k, v, _ = dev.read(None, [n], table[:1].cpu().numpy(), 0, 1, n, 0.0)
    cache.pool[...] = dev.pool()
    x = torch.randn((m, q_heads * d), device="cuda:0", generator=gen)
    x *= torch.exp(0.6 * torch.randn((m, 1), device="cuda:0", generator=gen))
    x = x.cpu().numpy()
    pos = [n - 1 - 7 * r for r in range(m)]
    tab = table[:m].cpu().numpy()
    got = dev.attention(x, pos, tab, 0, q_heads, n).reshape(m, kvh, -1, d)
    got_run = dev.attention(x, pos, tab, 0, q_heads, n, [(0, m)]).reshape(m, kvh, -1, d)
    # Values from codes and scales in 64 bits: read() has rounded their product.
    t = np.arange(n)
    page = tab[0, t // 16]
    f = Cache.floats(cache.pool)[page, 0, :, 0]                      # [tokens][kv heads][floats]
    rec = cache.pool[page, 0, :, 0]
    at_k = np.stack([cache.k_at(i) for i in range(16)])[t % 16][:, None]
    at_v = np.stack([cache.v_at(i) for i in range(16)])[t % 16][:, None]
    k64 = kv8_model.value(np.take_along_axis(rec, at_k, 2), kind) * f[..., 0:1].astype(np.float64)
    v64 = kv8_model.value(np.take_along_axis(rec, at_v, 2), kind) * f[..., 1:2].astype(np.float64)
    assert np.abs(k64.reshape(1, 1, n, -1) - k).max() <= 2.0 ** -24 * np.abs(k64).max()
    assert np.abs(v64.reshape(1, 1, n, -1) - v).max() <= 2.0 ** -24 * np.abs(v64).max()
    q = x.astype(np.float64).reshape(m, kvh, -1, d)
    want = np.empty(got.shape)
    for g in range(kvh):
        s = np.einsum("mhd,td->mht", q[:, g], k64[:, g]) / np.sqrt(d)
        s = np.where(np.arange(n)[None, None, :] > np.array(pos)[:, None, None], -np.inf, s)
        p = np.exp(s - s.max(axis=-1, keepdims=True))
        want[:, g] = np.einsum("mht,td->mhd", p / p.sum(axis=-1, keepdims=True), v64[:, g])
    for side in (got, got_run):
        err = np.linalg.norm(side - want) / np.linalg.norm(want)
        print("rms error in half steps of f32", err * 2 ** 24, flush=True)
        assert err <= 16 * 2.0 ** -24


@pytest.mark.gpu
@KINDS
def test_agrees_with_the_online_attention_over_read_values(torch_cuda, hip_ctx, kind):
    """The values read into an fp32 pool and attended to by
    air_hip_attention_online give the same rows."""
    torch = torch_cuda
    rng = np.random.default_rng(31)
    q_heads, kvh, d, page_tokens = 28, 4, 128, 16
    lengths = [130, 17, 400]
    cache, tables = _filled(kind, kvh, d, page_tokens, lengths, rng, layers=1, layer=0)
    dev = Device(torch, hip_ctx, cache)
    top = cache.max_pages * page_tokens
    k, v, _ = dev.read(None, lengths, tables, 0, 1, top, 0.0)
    pool = np.zeros((3 * cache.max_pages, 1, 2, page_tokens, kvh * d), dtype=np.float32)
    pool[:, 0, 0] = k.reshape(-1, page_tokens, kvh * d)
    pool[:, 0, 1] = v.reshape(-1, page_tokens, kvh * d)
    x = rows(rng, 3, q_heads, kvh, d)
    pos = [n - 1 for n in lengths]
    pool_d, x_d = dev.up(pool), dev.up(x)
    f32 = capi.KvLayout(pool_d.data_ptr(), page_tokens, kvh * d, 1, cache.max_pages, 3 * cache.max_pages)
    flat = dev.up(np.arange(3 * cache.max_pages, dtype=np.int32).reshape(3, -1))
    tiles = capi.attention_tiles([1, 1, 1], q_heads, kvh)
    tiles_d = dev.up(np.array(tiles, dtype=np.uint32).view(np.int32))
    pos_d = dev.up(pos, np.int32)
    out = torch.empty((3, q_heads * d), device="cuda:0")
    capi.check(dev.lib.air_hip_attention_online(hip_ctx.handle, ctypes.byref(f32), x_d.data_ptr(), x.shape[1], 3,
                                                pos_d.data_ptr(), flat.data_ptr(), 0, q_heads, kvh, d,
                                                tiles_d.data_ptr(), len(tiles), max(lengths), out.data_ptr()))
    got = dev.attention(x, pos, tables, 0, q_heads, max(lengths))
    want, tol, _ = cache.attention(x, pos, tables, 0, q_heads, max(lengths))
    # The other side has rounded code * scale to f32 (2^-24 of each value) as well.
    within(out.cpu().numpy(), got, 2 * tol + 2.0 ** -22 * np.abs(want).max())


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kvh,d,page_tokens,lengths,first,last,budget", [
    (4, 128, 16, [300, 64, 65, 0, 1], 4, 16, 64),
    (2, 64, 48, [500, 33, 129], 0, 0, 100),
    (1, 64, 16, [37, 21, 20], 10, 10, 20),            # nothing between is kept
    (3, 128, 32, [90, 700], 0, 1, 1),
])
def test_evict(torch_cuda, hip_ctx, kind, in_place, kvh, d, page_tokens, lengths, first, last, budget):
    """Kept slots and the bytes of the shortened pages equal the model's, with
    equal weights, NaN and negative ones, and a token without a page."""
    rng = np.random.default_rng(budget + kind)
    layers = 3
    max_pages = -(-max(lengths) // page_tokens) + 1
    pool = 2 * sum(-(-n // page_tokens) + 8 for n in lengths) + 4
    cache = Cache(kind, kvh, d, layers, page_tokens, pool, max_pages, seed=9)
    if kind == E4M3:
        codes = cache.pool[..., 128:]
        codes[(codes & 127) == 127] = 0
    both = page_tables(rng, lengths + [min(n, budget) for n in lengths], page_tokens, max_pages, pool)
    tables, new = both[:len(lengths)], both[len(lengths):]
    w = Cache.floats(cache.pool)[..., 16:32]
    w[...] = rng.integers(0, 6, w.shape).astype(np.float32) * np.float32(0.25)   # many ties
    w[..., 3] = np.nan
    w[..., 7] *= -1.0                                  # -0 and below
    w[0] = rng.exponential(1.0, w[0].shape).astype(np.float32)
    Cache.floats(cache.pool)[tables[0, 0], 1, 0, 0, 0] = np.nan     # a poisoned K block
    if lengths[0] > 5 * page_tokens:
        tables[0, 2] = -1
    if in_place:
        new = tables
    dev = Device(torch_cuda, hip_ctx, cache)
    top = max(lengths)
    got = dev.evict(lengths, tables, new, 1, 2, first, last, budget, top)
    want = cache.evict(lengths, tables, new, 1, 2, first, last, budget, top)
    assert np.array_equal(got, want)
    # Behind a shortened sequence's last token a block's slots hold nothing.
    pool_d = dev.pool()
    for i, n in enumerate(lengths):
        n = min(n, budget)
        for layer in (1, 2):
            for g in range(kvh):
                for t in range(n):
                    a = cache.token(new[i], layer, g, t)
                    at = cache.slot(new[i], layer, g, t)
                    if at is None:
                        continue
                    rec = pool_d[new[i][t // page_tokens], layer, g, t % page_tokens // 16]
                    assert np.array_equal(rec[cache.k_at(t % 16)], at[0][cache.k_at(t % 16)])
                    assert np.array_equal(rec[cache.v_at(t % 16)], at[0][cache.v_at(t % 16)])
                    assert same(rec.view(np.float32)[[0, 1, 16 + t % 16]], Cache.floats(at[0])[[0, 1, 16 + t % 16]])
                    assert a is not None
    assert same(pool_d[:, 0], cache.pool[:, 0])        # a layer that was not named


@pytest.mark.gpu
def test_evict_counts_up_to_max_tokens(torch_cuda, hip_ctx):
    """A length past max_tokens counts as max_tokens."""
    rng = np.random.default_rng(3)
    cache, tables = _filled(I8, 1, 64, 16, [200], rng, layers=1, layer=0)
    Cache.floats(cache.pool)[..., 16:32] = rng.exponential(1.0, cache.pool.shape[:-1] + (16,))
    dev = Device(torch_cuda, hip_ctx, cache)
    got = dev.evict([200], tables, tables, 0, 1, 2, 3, 40, 100)
    want = cache.evict([200], tables, tables, 0, 1, 2, 3, 40, 100)
    assert np.array_equal(got, want) and got.max() == 99


@pytest.mark.gpu
@KINDS
def test_serving_run(torch_cuda, hip_ctx, kind):
    """Two prompts appended and attended to in one call, their last rows
    setting the weights; decode steps that add to them; an eviction in place;
    decode steps that go on in the shortened cache.  Every step against the
    model."""
    rng = np.random.default_rng(41 + kind)
    q_heads, kvh, d, page_tokens, layers = 14, 2, 64, 16, 2
    prompts = [90, 61]
    cache = Cache(kind, kvh, d, layers, page_tokens, 30, 8, seed=5)
    tables = page_tables(rng, [128, 128], page_tokens, 8, 30)
    dev = Device(torch_cuda, hip_ctx, cache)
    qw = q_heads * d

    def step(named, runs, mode):
        pos, tab = [p for _, p in named], tables[[s for s, _ in named]]
        for layer in range(layers):
            x = rows(rng, len(named), q_heads, kvh, d)
            dev.append(x, qw, pos, tab, layer)
            cache.append(x, qw, pos, tab, layer)
            code = {None: 0, "add": 1, "set": 2}[mode]
            got = dev.attention(x, pos, tab, layer, q_heads, 128, runs, weights=code)
            want, tol, far = cache.attention(x, pos, tab, layer, q_heads, 128, runs, weights=mode)
            within(got, want, tol)
            pool = dev.pool()
            check_weights(cache, pool, far)
            assert np.array_equal(pool[..., 128:], cache.pool[..., 128:])
            cache.pool[...] = pool

    step([(0, p) for p in range(90)] + [(1, p) for p in range(61)], [(0, 90), (90, 151)], "set")
    lengths = prompts
    for _ in range(3):
        step([(0, lengths[0]), (1, lengths[1])], None, "add")
        lengths = [n + 1 for n in lengths]
    got = dev.evict(lengths, tables, tables, 0, layers, 4, 20, 64, 128)
    want = cache.evict(lengths, tables, tables, 0, layers, 4, 20, 64, 128)
    assert np.array_equal(got, want)
    assert same(dev.pool()[..., :128], cache.pool[..., :128]) or lengths[1] <= 64
    cache.pool[...] = dev.pool()
    lengths = [min(n, 64) for n in lengths]
    for _ in range(3):
        step([(0, lengths[0]), (1, lengths[1])], None, "add")
        lengths = [n + 1 for n in lengths]


@pytest.mark.gpu
def test_captured_steps_replay(torch_cuda):
    """Append and attention with weights, captured once and replayed over
    changed inputs, with eager work between the replays; two graphs of one
    context; each replay equals the eager calls on a copy of the cache."""
    torch = torch_cuda
    rng = np.random.default_rng(51)
    q_heads, kvh, d, page_tokens = 28, 4, 128, 16
    lengths = [600, 40, 333]
    cache, tables = _filled(I8, kvh, d, page_tokens, lengths, rng, layers=1, layer=0, max_pages=64)
    stream = torch.cuda.Stream()
    with capi.Context(0, stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        dev, ref = Device(torch, ctx, cache), Device(torch, ctx, cache)
        x = dev.up(rows(rng, 3, q_heads, kvh, d))
        pos = dev.up([n - 1 for n in lengths], np.int32)
        tab = dev.up(tables, np.int32)
        outs = [torch.zeros((3, q_heads * d), device="cuda:0") for _ in range(3)]

        def step(side, out, bound):
            capi.check(side.lib.air_hip_kv8_append(ctx.handle, ctypes.byref(side.kv), x.data_ptr(), x.shape[1],
                                                   q_heads * d, 3, pos.data_ptr(), tab.data_ptr(), 0))
            capi.check(side.lib.air_hip_kv8_attention(ctx.handle, ctypes.byref(side.kv), x.data_ptr(), x.shape[1], 3,
                                                      pos.data_ptr(), tab.data_ptr(), 0, q_heads, None, 0, bound,
                                                      capi.KV8_WEIGHTS_ADD, out.data_ptr()))
        for side in (dev, ref):
            step(side, outs[0], 1024)                 # sizes the scratch
        torch.cuda.synchronize()
        graphs = []
        for bound, out in ((1024, outs[0]), (700, outs[1])):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                step(dev, out, bound)
            graphs.append((g, out, bound))
        for i in range(6):
            g, out, bound = graphs[i % 2]
            x.copy_(dev.up(rows(rng, 3, q_heads, kvh, d)))
            pos.add_(1)
            torch.cuda.synchronize()
            g.replay()
            step(ref, outs[2], bound)
            torch.cuda.synchronize()
            assert torch.equal(out, outs[2]), i
            assert np.array_equal(dev.pool(), ref.pool()), i
    torch.cuda.synchronize()


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("q_heads,kvh,d,page_tokens,seqs", [
    (14, 2, 128, 16, [(0, 400), (300, 101)]),
    (6, 6, 64, 32, [(0, 331), (50, 90), (7, 1)]),
])
def test_large_prompts(torch_cuda, hip_ctx, kind, q_heads, kvh, d, page_tokens, seqs):
    """Runs long enough for tiles of several rows without weights too; eight
    rows at a time see the same tokens."""
    rng = np.random.default_rng(131 + q_heads + kind)
    lengths = [a + b + 8 for a, b in seqs]
    cache, tables = _filled(kind, kvh, d, page_tokens, lengths, rng, layers=1, layer=0)
    dev = Device(torch_cuda, hip_ctx, cache)
    pos, tab, runs = [], [], []
    for i, (a, b) in enumerate(seqs):
        runs.append((len(pos), len(pos) + b))
        pos += [a + r // 8 * 8 + 5 for r in range(b)]
        tab += [tables[i]] * b
    tab = np.array(tab)
    x = rows(rng, len(pos), q_heads, kvh, d)
    got = dev.attention(x, pos, tab, 0, q_heads, max(lengths), runs)
    want, tol, _ = cache.attention(x, pos, tab, 0, q_heads, max(lengths), runs)
    within(got, want, tol)


@pytest.mark.gpu
@KINDS
def test_many_runs(torch_cuda, hip_ctx, kind):
    """Seventy runs of one to nine rows (and empty ones), more than a wave
    looks up at a time; forty q heads of one KV head, so two parts of a tile."""
    rng = np.random.default_rng(61 + kind)
    q_heads, kvh, d, page_tokens = 40, 1, 64, 16
    rows_of = [int(n) for n in rng.integers(1, 10, 70)]
    before = [int(n) for n in rng.integers(0, 30, 70)]
    lengths = [a + b for a, b in zip(before, rows_of)]
    cache, tables = _filled(kind, kvh, d, page_tokens, lengths, rng, layers=1, layer=0)
    dev = Device(torch_cuda, hip_ctx, cache)
    pos, tab, runs = [], [], []
    for i, (a, b) in enumerate(zip(before, rows_of)):
        runs.append((len(pos), len(pos) + b))
        if i % 9 == 0:
            runs.append((len(pos) + b, len(pos) + b))
        pos += range(a, a + b)
        tab += [tables[i]] * b
    pos[runs[5][0]:runs[5][1]] = [-1] * (runs[5][1] - runs[5][0])     # a run that attends to nothing
    tab = np.array(tab)
    for mode, name in ((capi.KV8_WEIGHTS_NONE, None), (capi.KV8_WEIGHTS_SET, "set"), (capi.KV8_WEIGHTS_ADD, "add")):
        x = rows(rng, len(pos), q_heads, kvh, d)
        got = dev.attention(x, pos, tab, 0, q_heads, max(lengths), runs, weights=mode)
        want, tol, far = cache.attention(x, pos, tab, 0, q_heads, max(lengths), runs, weights=name)
        within(got, want, tol)
        pool = dev.pool()
        check_weights(cache, pool, far)
        cache.pool[...] = pool


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("kvh,d", [(8, 128), (8, 64)])
def test_tiles_past_a_full_card(torch_cuda, hip_ctx, kind, kvh, d):
    """More tiles than run at a time: those that fill the card are not cut,
    the ones left over are."""
    rng = np.random.default_rng(71 + kind)
    group, n = 16, 1090
    q_heads, m = kvh * group, 131 if d == 128 else 201
    cache, tables = _filled(kind, kvh, d, 16, [n, n + 7], rng, layers=1, layer=0)
    dev = Device(torch_cuda, hip_ctx, cache)
    cutoff = m // 2 + 3
    runs = [(0, cutoff), (cutoff, m)]
    tab = np.array([tables[0]] * cutoff + [tables[1]] * (m - cutoff))
    pos = [n - 1 - 300 * (r % 3) for r in range(m)]
    x = rows(rng, 6, q_heads, kvh, d)[np.arange(m) % 6]           # six rows over and over
    got = dev.attention(x, pos, tab, 0, q_heads, n + 7, runs)
    some = [r for start in (0, cutoff) for r in range(start, start + 6)]
    want, tol, _ = cache.attention(x[some], [pos[r] for r in some], tab[some], 0, q_heads, n + 7)
    like = [some.index(next(s for s in some if s % 6 == r % 6 and (s < cutoff) == (r < cutoff))) for r in range(m)]
    within(got, want[like], tol[like])


@pytest.mark.gpu
@KINDS
def test_runs_of_one_row_over_split_keys(torch_cuda, hip_ctx, kind):
    """Runs of a row each, one empty, one shorter than a split, over keys long
    enough to be cut, with weights: the launch that joins the splits takes the
    runs' rows."""
    rng = np.random.default_rng(81 + kind)
    q_heads, kvh, d = 12, 2, 64
    lengths = [2500, 30, 1200]
    cache, tables = _filled(kind, kvh, d, 32, lengths, rng, layers=1, layer=0)
    dev = Device(torch_cuda, hip_ctx, cache)
    pos, runs = [n - 1 for n in lengths], [(0, 1), (1, 1), (1, 2), (2, 3)]
    for mode, name in ((capi.KV8_WEIGHTS_ADD, "add"), (capi.KV8_WEIGHTS_SET, "set")):
        x = rows(rng, 3, q_heads, kvh, d, pad=8)
        got = dev.attention(x, pos, tables, 0, q_heads, 2500, runs, weights=mode)
        want, tol, far = cache.attention(x, pos, tables, 0, q_heads, 2500, runs, weights=name)
        within(got, want, tol)
        pool = dev.pool()
        check_weights(cache, pool, far)
        cache.pool[...] = pool


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("d", [64, 128])
def test_many_splits(torch_cuda, hip_ctx, kind, d):
    """Keys cut into more splits than one thread joins: single rows, one of
    them short, and a run, without weights and with."""
    rng = np.random.default_rng(141 + d + kind)
    q_heads, kvh, n = 3, 1, 9100
    cache, tables = _filled(kind, kvh, d, 64, [n, 100], rng, layers=1, layer=0)
    dev = Device(torch_cuda, hip_ctx, cache)
    single = ([n - 1, 99], tables, None)
    run = ([n - 1 - 290 * (r % 3) for r in range(30)], np.repeat(tables[:1], 30, axis=0), [(0, 30)])
    for pos, tab, runs in (single, run):
        for mode, name in ((capi.KV8_WEIGHTS_NONE, None), (capi.KV8_WEIGHTS_SET, "set")):
            x = rows(rng, len(pos), q_heads, kvh, d)
            got = dev.attention(x, pos, tab, 0, q_heads, n, runs, weights=mode)
            want, tol, far = cache.attention(x, pos, tab, 0, q_heads, n, runs, weights=name)
            within(got, want, tol)
            pool = dev.pool()
            check_weights(cache, pool, far)
            cache.pool[...] = pool


@pytest.mark.gpu
def test_runs_that_share_pages_add_up(torch_cuda, hip_ctx):
    """Two runs over one sequence's pages: what both add to a weight is
    there, whichever comes first (each addition rounds once)."""
    rng = np.random.default_rng(91)
    q_heads, kvh, d, n = 8, 2, 64, 200
    cache, tables = _filled(I8, kvh, d, 16, [n], rng, layers=1, layer=0)
    dev = Device(torch_cuda, hip_ctx, cache)
    pos = list(range(n - 8, n)) + list(range(n - 6, n))
    tab = np.repeat(tables, len(pos), axis=0)
    x = rows(rng, len(pos), q_heads, kvh, d)
    dev.attention(x, pos, tab, 0, q_heads, n, [(0, 8), (8, 14)], weights=capi.KV8_WEIGHTS_ADD)
    _, _, first = cache.attention(x[:8], pos[:8], tab[:8], 0, q_heads, n, [(0, 8)], weights="add")
    _, _, both = cache.attention(x[8:], pos[8:], tab[8:], 0, q_heads, n, [(0, 6)], weights="add")
    check_weights(cache, dev.pool(), [b[:4] + (a[4] + b[4],) for a, b in zip(first, both)])


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("kvh,d,budget", [(2, 128, 333), (1, 64, 400)])
def test_evict_many_blocks_in_place(torch_cuda, hip_ctx, kind, kvh, d, budget):
    """More blocks than a workgroup takes at a time, kept tokens crowded at
    the end (every block's sources lie far ahead) or at the front (a block is
    its own source)."""
    rng = np.random.default_rng(budget + kind)
    lengths = [900, 500, budget + 1]
    cache, tables = _filled(kind, kvh, d, 16, lengths, rng, layers=1, layer=0)
    for i, n in enumerate(lengths):
        for t in range(n):
            at = cache.slot(tables[i], 0, 0, t)
            for g in range(kvh):
                rec = cache.slot(tables[i], 0, g, t)[0]
                cache.floats(rec)[16 + at[1]] = np.float32(t if i == 0 else -t if i == 1 else rng.random())
    dev = Device(torch_cuda, hip_ctx, cache)
    got = dev.evict(lengths, tables, tables, 0, 1, 1, 2, budget, 900)
    want = cache.evict(lengths, tables, tables, 0, 1, 1, 2, budget, 900)
    assert np.array_equal(got, want)
    fill = 7.0
    for a, b in zip(dev.read(None, [budget] * 3, tables, 0, 1, budget, fill),
                    cache.read(None, [budget] * 3, tables, 0, 1, budget, fill)):
        assert np.array_equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_of_a_long_sequence(torch_cuda, hip_ctx, in_place):
    """More tokens than the selection holds in LDS, with equal weights on both
    sides of that bound."""
    rng = np.random.default_rng(121)
    n, budget = 17001, 700
    cache = Cache(I8, 1, 64, 1, 64, 290, 280, seed=8)
    Cache.floats(cache.pool)[..., 16:32] = rng.integers(0, 40, cache.pool.shape[:-1] + (16,))
    both = page_tables(rng, [n, budget], 64, 280, 290)
    tables = both[:1]
    new = tables if in_place else both[1:]
    dev = Device(torch_cuda, hip_ctx, cache)
    got = dev.evict([n], tables, new, 0, 1, 3, 30, budget, 280 * 64)
    want = cache.evict([n], tables, new, 0, 1, 3, 30, budget, 280 * 64)
    assert np.array_equal(got, want)
    for a, b in zip(dev.read(None, [budget], new, 0, 1, budget, 7.0), cache.read(None, [budget], new, 0, 1, budget, 7.0)):
        assert np.array_equal(a, b)


@pytest.mark.gpu
def test_two_contexts_at_once(torch_cuda):
    """Two contexts on two streams, their calls in turn without waiting:
    each result is that of its calls alone."""
    torch = torch_cuda
    rng = np.random.default_rng(101)
    q_heads, kvh, d = 14, 2, 64
    lengths = [700, 90]
    cache, tables = _filled(E4M3, kvh, d, 16, lengths, rng, layers=1, layer=0, max_pages=60)
    xs = [rows(rng, 2, q_heads, kvh, d) for _ in range(8)]

    def calls(dev, ctx, x, pos, tab, out):
        capi.check(dev.lib.air_hip_kv8_append(ctx.handle, ctypes.byref(dev.kv), x.data_ptr(), x.shape[1], q_heads * d,
                                              2, pos.data_ptr(), tab.data_ptr(), 0))
        capi.check(dev.lib.air_hip_kv8_attention(ctx.handle, ctypes.byref(dev.kv), x.data_ptr(), x.shape[1], 2,
                                                 pos.data_ptr(), tab.data_ptr(), 0, q_heads, None, 0, 960,
                                                 capi.KV8_WEIGHTS_ADD, out.data_ptr()))
        pos.add_(1)

    def run(together):
        streams = [torch.cuda.Stream() for _ in range(2)]
        ctxs = [capi.Context(0, s.cuda_stream) for s in streams]
        devs = [Device(torch, c, cache) for c in ctxs]
        sides = []
        for i, dev in enumerate(devs):
            sides.append((dev.up(np.array(lengths) + 3 * i, np.int32), dev.up(tables, np.int32),
                          [dev.up(x) for x in xs[4 * i:4 * i + 4]],
                          [torch.zeros((2, q_heads * d), device="cuda:0") for _ in range(4)]))
        torch.cuda.synchronize()
        order = [(i, j) for j in range(4) for i in range(2)] if together else [(i, j) for i in range(2) for j in range(4)]
        for i, j in order:
            pos, tab, x, out = sides[i]
            with torch.cuda.stream(streams[i]):
                calls(devs[i], ctxs[i], x[j], pos, tab, out[j])
            if not together:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        result = [torch.stack(s[3]).cpu().numpy() for s in sides] + [dev.pool() for dev in devs]
        for c in ctxs:
            c.close()
        return result

    together, alone = run(True), run(False)
    assert np.isfinite(together[0]).all()
    for a, b in zip(together, alone):                 # side 1 counts three stale slots as held: NaN codes among them
        assert np.array_equal(a, b, equal_nan=a.dtype == np.float32)


@pytest.mark.gpu
def test_captured_prompt_replays(torch_cuda):
    """A prompt's runs appended and attended to with weights, then an eviction
    to other pages, in one graph: replays over changed rows equal the eager
    calls, with a larger eager call (which regrows the scratch) between."""
    torch = torch_cuda
    rng = np.random.default_rng(111)
    q_heads, kvh, d, m = 14, 2, 64, 60
    cache = Cache(I8, kvh, d, 1, 16, 80, 20, seed=6)
    both = page_tables(rng, [300, 300, 48, 48], 16, 20, 80)
    stream = torch.cuda.Stream()
    with capi.Context(0, stream.cuda_stream) as ctx, torch.cuda.stream(stream):
        dev, ref = Device(torch, ctx, cache), Device(torch, ctx, cache)
        x = dev.up(rows(rng, m, q_heads, kvh, d))
        pos = dev.up(list(range(40, 70)) + list(range(100, 130)), np.int32)
        tab = dev.up(np.repeat(both[:2], 30, axis=0), np.int32)
        old, new, starts = dev.up(both[:2], np.int32), dev.up(both[2:], np.int32), dev.up([0, 30, 60], np.int32)
        lengths = dev.up([70, 130], np.int32)
        outs = [torch.zeros((m, q_heads * d), device="cuda:0") for _ in range(2)]
        kept = [torch.zeros(2 * kvh * 48, dtype=torch.int32, device="cuda:0") for _ in range(2)]

        def step(side, i, bound=320):
            lib, h, kv = side.lib, ctx.handle, ctypes.byref(side.kv)
            capi.check(lib.air_hip_kv8_append(h, kv, x.data_ptr(), x.shape[1], q_heads * d, m, pos.data_ptr(),
                                              tab.data_ptr(), 0))
            capi.check(lib.air_hip_kv8_attention(h, kv, x.data_ptr(), x.shape[1], m, pos.data_ptr(), tab.data_ptr(), 0,
                                                 q_heads, starts.data_ptr(), 2, bound, capi.KV8_WEIGHTS_ADD,
                                                 outs[i].data_ptr()))
            capi.check(lib.air_hip_kv8_evict(h, kv, 2, lengths.data_ptr(), old.data_ptr(), new.data_ptr(), 0, 1, 2, 8,
                                             48, 320, kept[i].data_ptr()))
        step(dev, 0)
        step(ref, 1)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step(dev, 0)
        wide = torch.zeros((4 * m, x.shape[1]), device="cuda:0")
        gone = torch.full((4 * m,), -1, dtype=torch.int32, device="cuda:0")
        wide_tab, wide_out = tab.repeat(4, 1), torch.empty((4 * m, q_heads * d), device="cuda:0")
        for i in range(4):
            x.copy_(dev.up(rows(rng, m, q_heads, kvh, d)))
            if i == 2:                                # rows that attend to nothing, more of them than before
                capi.check(dev.lib.air_hip_kv8_attention(ctx.handle, ctypes.byref(dev.kv), wide.data_ptr(), wide.shape[1],
                                                         4 * m, gone.data_ptr(), wide_tab.data_ptr(), 0, q_heads, None,
                                                         0, 320, capi.KV8_WEIGHTS_ADD, wide_out.data_ptr()))
            torch.cuda.synchronize()
            g.replay()
            step(ref, 1)
            torch.cuda.synchronize()
            assert torch.equal(outs[0], outs[1]) and torch.equal(kept[0], kept[1]), i
            assert np.array_equal(dev.pool(), ref.pool()), i
        assert not wide_out.any()
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_sizes_past_the_grids_are_refused(torch_cuda, hip_ctx):
    torch = torch_cuda
    lib, h = capi.lib(), hip_ctx.handle
    buf = torch.zeros(1 << 12, device="cuda:0")
    ints = torch.zeros(64, dtype=torch.int32, device="cuda:0")
    p, i = buf.data_ptr(), ints.data_ptr()

    def attend(kv_heads, heads, m, top):
        kv = capi.Kv8Layout(p, 16, kv_heads, 64, 1, 1 << 24, 1, None, 0, I8)
        return lib.air_hip_kv8_attention(h, ctypes.byref(kv), p, heads * 64, m, i, i, 0, heads, None, 0, top, 0, p)
    assert attend(65, 65, 65535, 16) == 6 and b"2^22" in lib.air_hip_last_error()
    assert attend(1, 1, 0, (1 << 27) + 1) == 6 and b"2^27" in lib.air_hip_last_error()
    assert attend(32, 32, 0, 1 << 27) == 6
    assert attend(16, 16, 0, 1 << 27) == 0
    kv = capi.Kv8Layout(p, 16, 1, 64, 1, 1 << 24, 1, None, 0, I8)
    for width in (2 ** 64 - 128, 2 ** 64 - 1, 400):   # the first two pass 2^64 with k and v
        assert lib.air_hip_kv8_append(h, ctypes.byref(kv), p, 512, width, 1, i, i, 0) == 1
    assert lib.air_hip_kv8_read(h, ctypes.byref(kv), 0, None, i, i, 0, 1, (1 << 27) + 1, p, None, None) == 6
    assert lib.air_hip_kv8_evict(h, ctypes.byref(kv), 0, i, i, i, 0, 1, 0, 0, 8, (1 << 27) + 1, i) == 6
    torch.cuda.synchronize()
    assert not buf.any() and not ints.any()


@pytest.mark.gpu
def test_refusals(torch_cuda, hip_ctx):
    """Every argument that the host can judge is refused with a message, and
    nothing runs."""
    torch = torch_cuda
    lib, h = capi.lib(), hip_ctx.handle
    buf = torch.zeros(1 << 16, device="cuda:0")
    ints = torch.zeros(64, dtype=torch.int32, device="cuda:0")
    p, i = buf.data_ptr(), ints.data_ptr()

    def layout(**over):
        f = dict(pool=p, page_tokens=16, kv_heads=2, head_dim=64, layers=2, max_pages=4, pool_pages=2, chunks=None,
                 chunk_shift=0, type=I8)
        f.update(over)
        return ctypes.byref(capi.Kv8Layout(*f.values()))

    def append(lay=None, x=p, stride=512, q_width=128, m=1, pos=i, tab=i, layer=0):
        return lib.air_hip_kv8_append(h, lay or layout(), x, stride, q_width, m, pos, tab, layer)

    def read(lay=None, seqs=1, lengths=i, tab=i, layer=0, layers=1, top=64, k=p):
        return lib.air_hip_kv8_read(h, lay or layout(), seqs, None, lengths, tab, layer, layers, top, k, None, None)

    def attend(lay=None, x=p, stride=512, m=1, pos=i, tab=i, layer=0, heads=4, starts=None, runs=0, top=64, mode=0,
               out=p + 4096):
        return lib.air_hip_kv8_attention(h, lay or layout(), x, stride, m, pos, tab, layer, heads, starts, runs, top,
                                         mode, out)

    def evict(lay=None, seqs=1, lengths=i, tab=i, new=i, layer=0, layers=1, first=0, last=0, budget=8, top=64, kept=i):
        return lib.air_hip_kv8_evict(h, lay or layout(), seqs, lengths, tab, new, layer, layers, first, last, budget,
                                     top, kept)

    bad_layouts = [dict(type=0), dict(type=7), dict(page_tokens=0), dict(page_tokens=20), dict(kv_heads=0),
                   dict(layers=0), dict(max_pages=0), dict(pool_pages=0), dict(pool=None), dict(pool=p + 8),
                   dict(pool_pages=2 ** 31), dict(chunks=i, chunk_shift=31), dict(chunks=i, chunk_shift=2)]
    for call in (append, read, attend, evict):
        for over in bad_layouts:
            assert call(lay=layout(**over)) == 1, (call.__name__, over)
            assert len(lib.air_hip_last_error()) > 0
        assert call(lay=layout(head_dim=96)) == 6 and b"64 and 128" in lib.air_hip_last_error()
        assert call(lay=layout(max_pages=2 ** 30)) == 6
        assert call(tab=None) == 1
    for over in [dict(x=None), dict(pos=None), dict(stride=383), dict(layer=2)]:
        assert append(**over) == 1, over
    for over in [dict(lengths=None), dict(layer=2), dict(layers=0), dict(layer=1, layers=2), dict(top=0), dict(top=65)]:
        assert read(**over) == 1, over
    assert read(seqs=65536) == 6
    for over in [dict(x=None), dict(pos=None), dict(out=None), dict(layer=2), dict(heads=0), dict(heads=3),
                 dict(top=0), dict(top=65), dict(mode=3), dict(mode=-1), dict(runs=1), dict(starts=i), dict(stride=255),
                 dict(stride=510), dict(x=p + 4), dict(out=p + 4)]:
        assert attend(**over) == 1, over
    for over in [dict(m=65536), dict(starts=i, runs=65536)]:
        assert attend(**over) == 6, over
    for over in [dict(lengths=None), dict(new=None), dict(kept=None), dict(layer=2), dict(layers=3), dict(budget=0),
                 dict(first=5, last=4), dict(first=2 ** 32 - 1, last=2), dict(top=0), dict(top=65)]:
        assert evict(**over) == 1, over
    assert evict(seqs=65536) == 6
    # Nothing to do is no error and touches nothing.
    assert append(m=0) == 0 and read(seqs=0) == 0 and attend(m=0) == 0 and evict(seqs=0) == 0
    torch.cuda.synchronize()
    assert not buf.any() and not ints.any()
