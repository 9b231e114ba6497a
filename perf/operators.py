"""The operators of the 8-bit KV cache, as measurable cases.

One pass is one use of the cache by a serving program, in its plain form (torch
operations in 32 bits) or through the entry points of air_amd.capi:

  append     quantise the k and v of one layer's q|k|v rows into their pages and
             read the touched blocks back;
  attention  the attention of one layer's rows over the cache, with the
             accumulated attention weights set and read back where the case
             says so;
  evict      keep the `budget` tokens of every sequence, layer and KV head that
             gathered the most weight, in new pages, and read those back.

Both forms work on the same pool.  A page is [layer][KV head][block] of records;
a record holds 16 tokens of one layer and KV head in 128 + 32 * head_dim bytes:

  0     f32 scale of K, f32 scale of V, 56 unused bytes
  64    f32 accumulated weight of each token
  128   K codes [token / 4][dim / 16][token % 4][dim % 16]
  ...   V codes [dim][token]

i8 codes are stored as code + 128, e4m3 codes as they are; a value is its code
times the block's scale.  Head counts and widths are those of the repository's
configurations (Qwen2-0.5B and Qwen2-7B) and generic ones.
"""
import ctypes
import math

import torch

own = False

BLOCK = 16          # tokens that share a scale
HEADER = 128        # bytes of a record before its codes
QMAX = {"i8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # A server's decode step stores one token of each sequence.
        dict(name="append_7b_tokens", kind="append", type="i8", heads=28, kv_heads=4, head_dim=128, page_tokens=16,
             layers=2, seqs=32, run=1, start_min=200, start_max=900),
        # A prompt quantum of two sequences that already hold some tokens.
        dict(name="append_7b_prompt", kind="append", type="e4m3", heads=28, kv_heads=4, head_dim=128, page_tokens=16,
             layers=2, seqs=2, run=509, start_min=0, start_max=37),
        # A token of a small model served alone: latency.
        dict(name="attention_05b_token", kind="attention", type="i8", heads=14, kv_heads=2, head_dim=64,
             page_tokens=16, layers=2, seqs=1, run=1, context_min=200, context_max=200, padded=0, weights=False),
        # A batched decode step in a graph of width 32, three rows of it padding.
        dict(name="attention_7b_batch", kind="attention", type="e4m3", heads=28, kv_heads=4, head_dim=128,
             page_tokens=16, layers=2, seqs=32, run=1, context_min=500, context_max=1200, padded=3, weights=False),
        # Decode over long ragged contexts.
        dict(name="attention_7b_long", kind="attention", type="i8", heads=28, kv_heads=4, head_dim=128,
             page_tokens=16, layers=1, seqs=24, run=1, context_min=700, context_max=4000, padded=0, weights=False),
        # A loaded server: the cache is far larger than the chip's own caches.
        dict(name="attention_server", kind="attention", type="i8", heads=32, kv_heads=8, head_dim=128,
             page_tokens=64, layers=1, seqs=48, run=1, context_min=4000, context_max=16000, padded=0, weights=False),
        # The first prompt quantum of a sequence.
        dict(name="attention_7b_prompt", kind="attention", type="i8", heads=28, kv_heads=4, head_dim=128,
             page_tokens=16, layers=1, seqs=1, run=512, context_min=512, context_max=512, padded=0, weights=False),
        # Later quanta of two long prompts, an odd number of rows.
        dict(name="attention_prompt_tail", kind="attention", type="e4m3", heads=28, kv_heads=4, head_dim=128,
             page_tokens=16, layers=1, seqs=2, run=301, context_min=3300, context_max=3801, padded=0, weights=False),
        # Decode that also notes which tokens are attended to.
        dict(name="weights_7b_batch", kind="attention", type="i8", heads=28, kv_heads=4, head_dim=128,
             page_tokens=16, layers=1, seqs=16, run=1, context_min=1000, context_max=3000, padded=0, weights=True),
        # The last rows of four prompts rank their tokens before an eviction.
        dict(name="weights_prompt_window", kind="attention", type="e4m3", heads=28, kv_heads=4, head_dim=128,
             page_tokens=16, layers=1, seqs=4, run=32, context_min=2900, context_max=4100, padded=0, weights=True),
        # One layer of one small model's sequence falls back to its budget.
        dict(name="evict_05b", kind="evict", type="e4m3", heads=14, kv_heads=2, head_dim=64, page_tokens=16, layers=2,
             seqs=1, context_min=1000, context_max=1000, keep_first=4, keep_last=64, budget=500),
        # Every layer of four long sequences, one of them within its budget.
        dict(name="evict_7b", kind="evict", type="i8", heads=28, kv_heads=4, head_dim=128, page_tokens=16, layers=6,
             seqs=4, context_min=900, context_max=4100, keep_first=4, keep_last=128, budget=1024),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    kind = rng.choice(["append", "attention", "attention", "prompt", "weights", "evict"])
    kv_heads = rng.choice([1, 2, 4, 8])
    case = dict(kind=kind, type=rng.choice(["i8", "e4m3"]), heads=kv_heads * rng.randint(1, 8), kv_heads=kv_heads,
                head_dim=rng.choice([64, 128]), page_tokens=16 * rng.choice([1, 1, 1, 2, 3, 4]),
                layers=rng.randint(1, 2))
    token_bytes = 2 * kv_heads * case["head_dim"]
    if kind == "append":
        run = _log_int(rng, 1, 512) if rng.random() < 0.5 else 1
        start = _log_int(rng, 1, 2000) - 1
        case.update(seqs=_log_int(rng, 1, max(1, min(64, 2048 // run))), run=run, start_min=start,
                    start_max=start + rng.randint(0, 50))
    elif kind == "evict":
        lo = _log_int(rng, 40, 4000)
        budget = _log_int(rng, 16, max(17, lo * 5 // 4))
        case.update(seqs=_log_int(rng, 1, 6), context_min=lo, context_max=lo + rng.randint(0, lo // 4),
                    keep_first=rng.randint(0, budget // 4), keep_last=rng.randint(0, budget // 3), budget=budget)
    else:
        case["kind"] = "attention"
        run = 1
        if kind == "prompt" or (kind == "weights" and rng.random() < 0.5):
            run = _log_int(rng, 2, 512)
        lo = max(run, _log_int(rng, 1, 6000))
        hi = lo + rng.randint(0, lo)
        most = min(48, 4.0e8 / (token_bytes * hi), 2.0e10 / (4.0 * case["head_dim"] * case["heads"] * run * hi))
        seqs = _log_int(rng, 1, max(1, int(most)))
        case.update(seqs=seqs, run=run, context_min=lo, context_max=hi,
                    padded=rng.randint(0, seqs // 4) if run == 1 else 0, weights=kind == "weights")
    return case


# ---- shapes -----------------------------------------------------------------

def _spread(case, lo, hi):
    """A value for each sequence, from lo to hi in a mixed order."""
    n = case["seqs"]
    return [lo + (hi - lo) * ((i * 7 + n - 1) % n) // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """Tokens each sequence holds; 0 for a padding row."""
    lens = _spread(case, case["context_min"], case["context_max"])
    pad = case.get("padded", 0)
    return lens[:len(lens) - pad] + [0] * pad if pad else lens


def _record(case):
    return HEADER + 2 * BLOCK * case["head_dim"]


def _max_pages(case, tokens):
    return -(-tokens // case["page_tokens"])


# ---- inputs -----------------------------------------------------------------

def _stored(x, kind):
    """Bytes and scale of blocks x [..., 16, D] of values: absmax / qmax in f32,
    quotients rounded to the nearest code."""
    scale = x.abs().amax(dim=(-2, -1)) / QMAX[kind]
    q = x / scale[..., None, None]
    if kind == "i8":
        return (q.round().clamp(-127, 127) + 128).to(torch.uint8), scale
    return q.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _fill(case, pages, gen):
    """A pool of `pages` pages whose every slot holds a token: pages that were
    in use before are what a server's pool consists of."""
    d, bpp = case["head_dim"], case["page_tokens"] // BLOCK
    lead = (pages, case["layers"], case["kv_heads"], bpp)
    pool = torch.empty(lead + (_record(case),), dtype=torch.uint8, device="cuda")
    at = max(1, (1 << 27) // max(1, math.prod(lead[1:]) * BLOCK * d))
    # Keys have channels that are larger everywhere, heads differ in size.
    channel = torch.exp(0.5 * torch.randn((case["layers"], case["kv_heads"], 1, 1, d), device="cuda", generator=gen))
    for p in range(0, pages, at):
        n = min(at, pages - p)
        shape = (n,) + lead[1:] + (BLOCK, d)
        k, ks = _stored(torch.randn(shape, device="cuda", generator=gen) * channel, case["type"])
        v, vs = _stored(torch.randn(shape, device="cuda", generator=gen), case["type"])
        w = torch.empty(shape[:-1], device="cuda").exponential_(1.0, generator=gen)
        rec = pool[p:p + n]
        rec[..., :HEADER] = 0
        rec[..., 0:4] = ks[..., None].view(torch.uint8)
        rec[..., 4:8] = vs[..., None].view(torch.uint8)
        rec[..., 64:128] = w.view(torch.uint8)
        k = k.reshape(shape[:-2] + (4, 4, d // 16, 16)).transpose(-3, -2)
        rec[..., HEADER:HEADER + BLOCK * d] = k.reshape(k.shape[:-4] + (-1,))
        rec[..., HEADER + BLOCK * d:] = v.transpose(-2, -1).reshape(shape[:-2] + (-1,))
    return pool


def _tables(case, tokens, gen, sets=1):
    """Page tables of `sets` times all sequences over one pool, in scattered
    order: [sets][seqs][max_pages], -1 past a sequence's own pages."""
    width = max(1, max(_max_pages(case, t) for t in tokens))
    need = [_max_pages(case, t) for t in tokens] * sets
    pages = max(1, sum(need))
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    held = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    tables = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    tables[held] = order[:sum(need)]
    return tables.view(sets, len(tokens), width), pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    d, width = case["head_dim"], case["kv_heads"] * case["head_dim"]
    state = dict(case=case)
    if case["kind"] == "evict":
        lens = _lengths(case)
        (old, new), pages = _tables(case, [max(t, case["budget"]) for t in lens], gen, sets=2)
        state.update(tables=old.contiguous(), new_tables=new.contiguous(), max_tokens=max(lens),
                     lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                     new_lengths=torch.tensor([min(t, case["budget"]) for t in lens], dtype=torch.int32, device="cuda"),
                     kept=torch.zeros((case["seqs"], case["layers"], case["kv_heads"], case["budget"]),
                                      dtype=torch.int32, device="cuda"))
        shape = (case["layers"], case["seqs"], case["budget"])
        state["pool"] = _fill(case, pages, gen)
        state["k"] = torch.zeros(shape + (width,), device="cuda")
        state["v"] = torch.zeros(shape + (width,), device="cuda")
        state["w"] = torch.zeros(shape + (case["kv_heads"],), device="cuda")
        return state
    run = case["run"]
    m = case["seqs"] * run
    if case["kind"] == "append":
        starts = _spread(case, case["start_min"], case["start_max"])
        lens = [s + run for s in starts]
        # Tokens read back of each sequence, at most: no more than a table names.
        back = min(-(-run // BLOCK) * BLOCK + BLOCK, _max_pages(case, max(lens)) * case["page_tokens"])
        lo = [s // BLOCK * BLOCK for s in starts]
        state.update(back=back, lo=torch.tensor(lo, dtype=torch.int32, device="cuda"),
                     count=torch.tensor([n - b for n, b in zip(lens, lo)], dtype=torch.int32, device="cuda"),
                     k=torch.zeros((case["seqs"], back, width), device="cuda"),
                     v=torch.zeros((case["seqs"], back, width), device="cuda"))
    else:
        lens = _lengths(case)
        starts = [n - run if n else -1 for n in lens]
        state.update(out=torch.zeros((m, case["heads"] * d), device="cuda"),
                     lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                     w=torch.zeros((case["seqs"], max(lens), case["kv_heads"]), device="cuda"))
    (tables,), pages = _tables(case, lens, gen)
    positions = torch.tensor(starts, dtype=torch.int32, device="cuda")[:, None] + torch.arange(
        run, dtype=torch.int32, device="cuda")[None, :]
    state.update(pool=_fill(case, pages, gen), tables=tables.contiguous(), positions=positions.reshape(-1).contiguous(),
                 row_tables=tables.repeat_interleave(run, dim=0).contiguous(), max_tokens=max(lens),
                 run_starts=torch.arange(0, m + 1, run, dtype=torch.int32, device="cuda"),
                 qkv=torch.randn((m, case["heads"] * d + 2 * width), device="cuda", generator=gen))
    # Queries as they meet keys: a few of them look hard at a few tokens.
    state["qkv"][:, :case["heads"] * d] *= torch.exp(0.5 * torch.randn((m, 1), device="cuda", generator=gen))
    return state


# ---- the plain form ---------------------------------------------------------

def _decode(codes, kind):
    if kind == "i8":
        return codes.float() - 128.0
    return codes.view(torch.float8_e4m3fn).float()


def _blocks(case, pool, tables, first, count):
    """Records of blocks first .. first + count - 1 of every sequence:
    [seqs][count][layers][kv_heads][record]; blocks without a page are zeros."""
    bpp = case["page_tokens"] // BLOCK
    block = first[:, None] + torch.arange(count, device="cuda")[None, :]
    slot = (block // bpp).clamp(max=tables.shape[1] - 1)
    page = torch.gather(tables, 1, slot).long()
    got = pool[page.clamp(min=0), :, :, (block % bpp)]
    return torch.where(((page >= 0) & (block // bpp < tables.shape[1]))[..., None, None, None], got, 0)


def _unpack(case, rec):
    """Codes' values [..., 16, D] of K and V, their scales and the weights."""
    d = case["head_dim"]
    k = rec[..., HEADER:HEADER + BLOCK * d].reshape(rec.shape[:-1] + (4, d // 16, 4, 16)).transpose(-3, -2)
    v = rec[..., HEADER + BLOCK * d:].reshape(rec.shape[:-1] + (d, BLOCK)).transpose(-2, -1)
    head = rec[..., :HEADER].contiguous().view(torch.float32)
    return (_decode(k.reshape(v.shape).contiguous(), case["type"]), head[..., 0],
            _decode(v.contiguous(), case["type"]), head[..., 1], head[..., 16:32])


def _round(q, kind):
    """Values of the nearest codes."""
    if kind == "i8":
        return q.round().clamp(-127, 127)
    return q.clamp(-448, 448).to(torch.float8_e4m3fn).float()


def _append_values(case, x, old, scale, written, held):
    """Values of blocks after storing x where `written`: all [seqs][blocks]
    [kv_heads][16][D], masks [seqs][blocks][16]."""
    mask = written[:, :, None, :, None]
    need = torch.where(mask, x, 0).abs().amax(dim=(-2, -1)) / QMAX[case["type"]]
    new = torch.where(held.any(dim=-1)[:, :, None], torch.maximum(scale, need), need)
    # A scale of zero holds zeros.
    inverse = torch.where(new > 0, new, 1)[..., None, None]
    moved = _round(old * (scale[..., None, None] / inverse), case["type"])
    kept = torch.where((new > scale)[..., None, None], moved, old)
    codes = torch.where(mask, _round(x / inverse, case["type"]), torch.where(held[:, :, None, :, None], kept, 0))
    return codes * new[..., None, None]


def _plain_append(state):
    case = state["case"]
    d, kvh, run = case["head_dim"], case["kv_heads"], case["run"]
    count = state["back"] // BLOCK
    start = state["positions"].view(case["seqs"], run)[:, 0]
    layer = case["layers"] - 1
    rec = _blocks(case, state["pool"], state["tables"], start // BLOCK, count)[:, :, layer]
    k, ks, v, vs, _ = _unpack(case, rec)
    token = state["lo"][:, None] + torch.arange(state["back"], device="cuda")[None, :]
    written = (token >= start[:, None]) & (token < start[:, None] + run)
    held = (token < start[:, None]).view(case["seqs"], count, BLOCK)
    row = (token - start[:, None]).clamp(0, run - 1).long()
    new = state["qkv"][:, case["heads"] * d:].view(case["seqs"], run, 2, kvh, d)
    new = torch.gather(new, 1, row[:, :, None, None, None].expand(-1, -1, 2, kvh, d))
    new = new.view(case["seqs"], count, BLOCK, 2, kvh, d).permute(3, 0, 1, 4, 2, 5)
    written = written.view(case["seqs"], count, BLOCK)
    live = (written | held).view(case["seqs"], -1, 1)
    back = [_append_values(case, x, old, s, written, held) for x, old, s in ((new[0], k, ks), (new[1], v, vs))]
    return [torch.where(live, b.permute(0, 1, 3, 2, 4).reshape(case["seqs"], -1, kvh * d), 0) for b in back]


def _plain_attention(state):
    case = state["case"]
    d, kvh, run, seqs = case["head_dim"], case["kv_heads"], case["run"], case["seqs"]
    group = case["heads"] // kvh
    blocks = -(-state["max_tokens"] // BLOCK)
    rec = _blocks(case, state["pool"], state["tables"], torch.zeros_like(state["lengths"]), blocks)
    k, ks, v, vs, _ = _unpack(case, rec[:, :, case["layers"] - 1])
    k = (k * ks[..., None, None]).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, d)
    v = (v * vs[..., None, None]).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, d)
    q = state["qkv"][:, :case["heads"] * d].reshape(seqs, run, kvh, group, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(seqs, kvh, run * group, d)
    s = torch.matmul(q, k.transpose(-2, -1).contiguous()) / math.sqrt(d)
    token = torch.arange(s.shape[-1], device="cuda")
    live = token <= state["positions"].view(seqs, run)[:, None, :, None, None].expand(-1, -1, -1, group, 1).reshape(
        seqs, 1, run * group, 1)
    s = torch.where(live, s, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0))
    total = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1)
    out = torch.matmul(p, v).reshape(seqs, kvh, run, group, d).permute(0, 2, 1, 3, 4).reshape(seqs * run, -1)
    if not case["weights"]:
        return out
    return [out, p.sum(dim=2).transpose(1, 2)[:, :state["max_tokens"]].contiguous()]


def _plain_evict(state):
    case = state["case"]
    d, kvh, seqs, budget = case["head_dim"], case["kv_heads"], case["seqs"], case["budget"]
    blocks = -(-state["max_tokens"] // BLOCK)
    rec = _blocks(case, state["pool"], state["tables"], torch.zeros_like(state["lengths"]), blocks)
    rec = rec.permute(0, 2, 3, 1, 4)                         # [seqs][layers][kv_heads][blocks][record]
    k, ks, v, vs, w = _unpack(case, rec)
    w = w.reshape(w.shape[:3] + (-1,))
    tokens = w.shape[-1]
    t = torch.arange(tokens, device="cuda")
    n = state["lengths"][:, None, None, None]
    rank = torch.where((t < case["keep_first"]) | (t >= n - case["keep_last"]), math.inf, w)
    rank = torch.where(t < n, rank, -math.inf)
    pick = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    pick = torch.sort(torch.where(pick < n, pick, tokens), dim=-1).values
    if pick.shape[-1] < budget:
        pick = torch.nn.functional.pad(pick, (0, budget - pick.shape[-1]), value=tokens)
    live = pick < n
    at = pick.clamp(max=tokens - 1)
    pad = -(-budget // BLOCK) * BLOCK - budget
    got = []
    for codes, scale in ((k, ks), (v, vs)):
        codes = torch.gather(codes.reshape(codes.shape[:3] + (-1, d)), 3, at[..., None].expand(at.shape + (d,)))
        scale = torch.where(live, torch.gather(scale, 3, at // BLOCK), 0)
        top = torch.nn.functional.pad(scale, (0, pad)).reshape(scale.shape[:3] + (-1, BLOCK)).amax(dim=-1)
        top = top.repeat_interleave(BLOCK, dim=-1)[..., :budget]
        codes = _round(codes * (scale / torch.where(top > 0, top, 1))[..., None], case["type"])
        value = torch.where(live[..., None], codes * top[..., None], 0)
        got.append(value.permute(1, 0, 3, 2, 4).reshape(case["layers"], seqs, budget, kvh * d))
    w = torch.where(live, torch.gather(w, 3, at), 0).permute(1, 0, 3, 2).contiguous()
    return [torch.where(live, pick, -1).to(torch.int32)] + got + [w]


# ---- the framework's calls --------------------------------------------------

_context = {}


def _handles(state):
    """The library, the context and the layout a program keeps."""
    from air_amd import capi

    if "ctx" not in _context:
        _context["ctx"] = capi.Context(0, torch.cuda.current_stream().cuda_stream)
    if "kv" not in state:
        case = state["case"]
        kinds = {"i8": capi.KV8_I8, "e4m3": capi.KV8_E4M3}
        state["kv"] = capi.Kv8Layout(state["pool"].data_ptr(), case["page_tokens"], case["kv_heads"],
                                     case["head_dim"], case["layers"], state["tables"].shape[1],
                                     state["pool"].shape[0], None, 0, kinds[case["type"]])
    return capi, capi.lib(), _context["ctx"].handle, ctypes.byref(state["kv"])


def _own_append(state):
    case = state["case"]
    capi, lib, ctx, kv = _handles(state)
    qkv, layer = state["qkv"], case["layers"] - 1
    capi.check(lib.air_hip_kv8_append(ctx, kv, qkv.data_ptr(), qkv.shape[1], case["heads"] * case["head_dim"],
                                      qkv.shape[0], state["positions"].data_ptr(), state["row_tables"].data_ptr(),
                                      layer))
    capi.check(lib.air_hip_kv8_read(ctx, kv, case["seqs"], state["lo"].data_ptr(), state["count"].data_ptr(),
                                    state["tables"].data_ptr(), layer, 1, state["back"], state["k"].data_ptr(),
                                    state["v"].data_ptr(), None))
    return [state["k"], state["v"]]


def _own_attention(state):
    case = state["case"]
    capi, lib, ctx, kv = _handles(state)
    qkv, layer = state["qkv"], case["layers"] - 1
    mode = capi.KV8_WEIGHTS_SET if case["weights"] else capi.KV8_WEIGHTS_NONE
    capi.check(lib.air_hip_kv8_attention(ctx, kv, qkv.data_ptr(), qkv.shape[1], qkv.shape[0],
                                         state["positions"].data_ptr(), state["row_tables"].data_ptr(), layer,
                                         case["heads"], state["run_starts"].data_ptr(), case["seqs"],
                                         state["max_tokens"], mode, state["out"].data_ptr()))
    if not case["weights"]:
        return state["out"]
    capi.check(lib.air_hip_kv8_read(ctx, kv, case["seqs"], None, state["lengths"].data_ptr(),
                                    state["tables"].data_ptr(), layer, 1, state["max_tokens"], None, None,
                                    state["w"].data_ptr()))
    return [state["out"], state["w"]]


def _own_evict(state):
    case = state["case"]
    capi, lib, ctx, kv = _handles(state)
    capi.check(lib.air_hip_kv8_evict(ctx, kv, case["seqs"], state["lengths"].data_ptr(), state["tables"].data_ptr(),
                                     state["new_tables"].data_ptr(), 0, case["layers"], case["keep_first"],
                                     case["keep_last"], case["budget"], state["max_tokens"],
                                     state["kept"].data_ptr()))
    capi.check(lib.air_hip_kv8_read(ctx, kv, case["seqs"], None, state["new_lengths"].data_ptr(),
                                    state["new_tables"].data_ptr(), 0, case["layers"], case["budget"],
                                    state["k"].data_ptr(), state["v"].data_ptr(), state["w"].data_ptr()))
    return [state["kept"], state["k"], state["v"], state["w"]]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "evict": _own_evict}[kind](state)
    return {"append": _plain_append, "attention": _plain_attention, "evict": _plain_evict}[kind](state)


# ---- what a pass cannot do without ------------------------------------------

def work(case):
    d, kvh = case["head_dim"], case["kv_heads"]
    token = kvh * (2 * d + 8 / BLOCK)                        # codes and scales of a token
    if case["kind"] == "append":
        m = case["seqs"] * case["run"]
        starts = _spread(case, case["start_min"], case["start_max"])
        read_back = m + sum(s % BLOCK for s in starts)
        return dict(bytes=m * 2 * kvh * d * 4 + m * token + read_back * 2 * kvh * d * 4, flops=0)
    lens = _lengths(case)
    if case["kind"] == "evict":
        rows = sum(min(n, case["budget"]) for n in lens) * case["layers"]
        weights = sum(lens) * case["layers"] * kvh * 4
        return dict(bytes=weights + rows * (2 * token + kvh * (2 * d * 4 + 4 + 4 + 4)), flops=0)
    rows = case["run"] * case["heads"] * d
    pairs = sum(sum(n - i for i in range(case["run"])) for n in lens if n)
    read = sum(lens) * token + case["seqs"] * rows * 8
    if case["weights"]:
        read += sum(lens) * kvh * 8
    return dict(bytes=read, flops=4 * d * case["heads"] * pairs)


# ---- the definition in 64 bits ----------------------------------------------

def _table(kind):
    """What each of the 256 codes stands for, in 64 bits."""
    if kind == "i8":
        return torch.arange(256, dtype=torch.float64) - 128
    values = []
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        x = math.nan if e == 15 and f == 7 else f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        values.append(-x if c & 128 else x)
    return torch.tensor(values, dtype=torch.float64)


def _near(q, kind):
    """The nearest code's value of f32 quotients, in 64 bits; ties to even."""
    q = q.double()
    if kind == "i8":
        return torch.round(q).clamp(-127, 127)
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(q / step) * step).clamp(-448, 448)


class _Sequence:
    """One sequence's tokens of one layer, as [tokens][kv_heads][D] codes in 64
    bits with the scale of each token's block."""

    def __init__(self, state, i, layer, tokens):
        case = state["case"]
        d, bpp = case["head_dim"], case["page_tokens"] // BLOCK
        pages = state["tables"][i, :_max_pages(case, tokens)].long()
        rec = state["pool"][pages, layer].transpose(0, 1).reshape(case["kv_heads"], len(pages) * bpp, -1)
        floats = rec.contiguous().view(torch.float32)
        lut = _table(case["type"]).to(rec.device)
        t = torch.arange(tokens, device=rec.device)
        at_k = HEADER + ((t % BLOCK) // 4 * (d // 16) * 64 + t % 4 * 16)[:, None] + (
            torch.arange(d, device=rec.device) // 16 * 64 + torch.arange(d, device=rec.device) % 16)[None, :]
        at_v = HEADER + BLOCK * d + torch.arange(d, device=rec.device)[None, :] * BLOCK + (t % BLOCK)[:, None]
        self.k = lut[rec[:, (t // BLOCK)[:, None], at_k].long()].transpose(0, 1)
        self.v = lut[rec[:, (t // BLOCK)[:, None], at_v].long()].transpose(0, 1)
        self.ks, self.vs = (floats[:, t // BLOCK, j].double().transpose(0, 1) for j in (0, 1))
        self.w = floats[:, t // BLOCK, 16 + t % BLOCK].transpose(0, 1)


def _exact_append(state):
    case = state["case"]
    d, kvh, run = case["head_dim"], case["kv_heads"], case["run"]
    outs = [torch.zeros((case["seqs"], state["back"], kvh, d), dtype=torch.float64, device="cuda") for _ in range(2)]
    rows = state["qkv"][:, case["heads"] * d:].view(case["seqs"], run, 2, kvh, d)
    for i in range(case["seqs"]):
        start = int(state["positions"][i * run])
        seq = _Sequence(state, i, case["layers"] - 1, start + run)
        lo = start // BLOCK * BLOCK
        for b in range(lo, start + run, BLOCK):
            first, last = max(b, start), min(b + BLOCK, start + run)
            for j, (codes, scale) in enumerate(((seq.k, seq.ks), (seq.v, seq.vs))):
                x = rows[i, first - start:last - start, j]                       # [tokens][kv_heads][D], f32
                need = x.abs().amax(dim=(0, 2)) / QMAX[case["type"]]
                old = scale[b].float()
                new = torch.maximum(old, need) if first > b else need
                held = codes[b:first]
                moved = _near(held.float() * (old / new)[None, :, None], case["type"])
                held = torch.where((new > old)[None, :, None], moved, held)
                block = torch.cat([held, _near(x / new[None, :, None], case["type"])])
                outs[j][i, b - lo:last - lo] = block * new.double()[None, :, None]
    return [o.view(case["seqs"], state["back"], -1) for o in outs]


def _exact_attention(state):
    case = state["case"]
    d, kvh, run = case["head_dim"], case["kv_heads"], case["run"]
    group = case["heads"] // kvh
    out = torch.zeros((case["seqs"] * run, kvh, group, d), dtype=torch.float64, device="cuda")
    weight = torch.zeros((case["seqs"], state["max_tokens"], kvh), dtype=torch.float64, device="cuda")
    q = state["qkv"][:, :case["heads"] * d].double().view(-1, kvh, group, d)
    lens = state["lengths"].tolist()
    for i, n in enumerate(lens):
        if n == 0:
            continue
        seq = _Sequence(state, i, case["layers"] - 1, n)
        pos = state["positions"][i * run:(i + 1) * run].long()
        late = torch.arange(n, device="cuda")[None, :] > pos[:, None]
        for g in range(kvh):
            k, v = seq.k[:, g] * seq.ks[:, g, None], seq.v[:, g] * seq.vs[:, g, None]
            for h in range(group):
                s = (q[i * run:(i + 1) * run, g, h] @ k.T) * d ** -0.5
                p = torch.softmax(s.masked_fill(late, -math.inf), dim=1)
                out[i * run:(i + 1) * run, g, h] = p @ v
                weight[i, :n, g] += p.sum(dim=0)
    out = out.view(case["seqs"] * run, -1)
    return [out, weight] if case["weights"] else out


def _exact_evict(state):
    case = state["case"]
    d, kvh, budget = case["head_dim"], case["kv_heads"], case["budget"]
    shape = (case["layers"], case["seqs"], budget, kvh)
    kept = torch.full((case["seqs"], case["layers"], kvh, budget), -1, dtype=torch.int32)
    outs = [torch.zeros(shape + (d,), dtype=torch.float64, device="cuda") for _ in range(2)]
    weight = torch.zeros(shape, dtype=torch.float64, device="cuda")
    lens = state["lengths"].tolist()
    for i, n in enumerate(lens):
        for layer in range(case["layers"]):
            seq = _Sequence(state, i, layer, n)
            ws = seq.w.cpu().tolist()
            for g in range(kvh):
                ids = list(range(n))
                if n > budget:
                    middle = list(range(case["keep_first"], n - case["keep_last"]))
                    middle.sort(key=lambda t: (-ws[t][g], t))
                    ids = sorted(list(range(case["keep_first"])) + list(range(n - case["keep_last"], n)) +
                                 middle[:budget - case["keep_first"] - case["keep_last"]])
                kept[i, layer, g, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
                at = torch.tensor(ids, device="cuda")
                weight[layer, i, :len(ids), g] = seq.w[at, g].double()
                for j, (codes, scale) in enumerate(((seq.k, seq.ks), (seq.v, seq.vs))):
                    own_scale = scale[at, g].float()
                    top = torch.cat([c.max().expand(len(c)) for c in own_scale.split(BLOCK)])
                    block = _near(codes[at, g].float() * (own_scale / top)[:, None], case["type"])
                    outs[j][layer, i, :len(ids), g] = block * top.double()[:, None]
    flat = [o.view(case["layers"], case["seqs"], budget, -1) for o in outs]
    return [kept.to("cuda")] + flat + [weight]


def exact(case, seed):
    """What run() returns for these inputs, from the definition in 64 bits (the
    stored codes and scales are the operator's, quotients in f32)."""
    state = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "evict": _exact_evict}[case["kind"]](state)
