"""Performance cases of a 4-bit cache held in pages that sequences share.

Keys and values are held in groups of 32 dims, 16 levels a group: step and lowest
value in half precision, so a slot of a 128-wide head takes 160 bytes for both.
Pages of some tens of slots belong to sequences through a table, with a count of the
entries that hold each page.  Rows are stored and read back (``pages_store``,
``pages_load``), queries attend over them (``attention_pages``), beams take over
their parents' pages and get copies of what they write (``pages_fork``,
``pages_reserve``), kept slots are moved together and the pages behind them given
back (``pages_compact``, ``pages_free``), and pages move between pools
(``pages_copy``).

Kinds: ``store`` (rows stored, then read back), ``attention``, ``beams`` (fork and
reserve), ``compact`` (reserve, compact, free) and ``copy``.  With ``own`` false,
``run`` computes a pass in elementary torch operations; with ``own`` true it calls
``kanjoos_amd``.  ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}
A3B = dict(n_head=32, n_head_kv=4, head_dim=128)
HEADS = [(32, 4, 128), (32, 4, 128), (32, 8, 128), (16, 4, 128), (12, 4, 128), (8, 8, 64), (8, 2, 64), (16, 2, 64)]
SHIFTS = [0, 16, 4, 20, 8, 24, 12, 28]  # of a word's eight codes


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # 32 sequences' new keys and values, read back as a draft model's fallback would
        dict(name="store_step", kind="store", type="f32", n_seq=32, rows=1, page=64, slots=2304, **A3B),
        # a prompt's keys and values
        dict(name="store_prompt", kind="store", type="f32", n_seq=1, rows=4096, page=64, slots=4352, **A3B),
        # one decode token at a short context: latency
        dict(name="step_1k", kind="attention", type="f32", n_seq=1, rows=1, prefix=1000, ragged=False, tree=False, page=64,
             **A3B),
        # a batch's decode step over long contexts
        dict(name="step_32x8k", kind="attention", type="bf16", n_seq=32, rows=1, prefix=8000, ragged=True, tree=False,
             page=64, **A3B),
        # a tree of drafts at the longest context
        dict(name="tree_25_32k", kind="attention", type="f16", n_seq=1, rows=25, prefix=32700, ragged=False, tree=True,
             page=128, **A3B),
        # a piece of a prompt behind a shared one: the most work
        dict(name="prompt_500_8k", kind="attention", type="bf16", n_seq=1, rows=500, prefix=8000, ragged=False, tree=False,
             page=64, **A3B),
        # a small beam search's step, all layers
        dict(name="beams_4", kind="beams", groups=1, beams=4, length=1000, tail=90, page=64, n_layer=48, n_head_kv=4,
             head_dim=128),
        # many answers a prompt for several prompts, in small pages
        dict(name="beams_8x4", kind="beams", groups=8, beams=4, length=4000, tail=200, page=16, n_layer=48, n_head_kv=4,
             head_dim=128),
        # the accepted paths of 32 sequences' drafts moved behind their prefixes
        dict(name="accept_32x8", kind="compact", n_seq=32, length=2048, tail=8, kept=0.5, page=64, n_layer=48, n_head_kv=4,
             head_dim=128),
        # half of a long context let go
        dict(name="evict_16k", kind="compact", n_seq=1, length=16000, tail=15996, kept=0.5, page=64, n_layer=48, n_head_kv=4,
             head_dim=128),
        # a short prompt's pages taken into another pool
        dict(name="copy_8", kind="copy", n=8, n_page=64, to_page=96, page=64, n_layer=48, n_head_kv=4, head_dim=128),
        # a whole pool moved into a larger one
        dict(name="copy_400", kind="copy", n=400, n_page=420, to_page=512, page=64, n_layer=48, n_head_kv=4, head_dim=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attention", "attention", "attention", "beams", "compact", "compact", "copy"])
    nh, nk, D = rng.choice(HEADS)
    heads = dict(n_head=nh, n_head_kv=nk, head_dim=D)
    page = rng.choice([16, 32, 64, 64, 128, 256])
    if kind == "store":
        n_seq = _log(rng, 1, 32)
        rows = _log(rng, 1, 4096 // n_seq)
        return dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), n_seq=n_seq, rows=rows, page=page,
                    slots=rows + rng.randint(1, 300), **heads)
    if kind == "attention":
        n_seq = rng.choice([1, 1, _log(rng, 2, 32)])
        rows = rng.choice([1, _log(rng, 1, 64), _log(rng, 1, 500)])
        most = min(32700, 500 * 32 * 8000 // (n_seq * rows * nh), 32 * 8000 // n_seq)
        return dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), n_seq=n_seq, rows=rows, prefix=_log(rng, 1, most),
                    ragged=rng.random() < 0.5, tree=rows <= 64 and rng.random() < 0.6, page=page, **heads)
    pool = dict(page=page, n_layer=rng.choice([8, 24, 48]), n_head_kv=nk, head_dim=D)
    per_slot = pool["n_layer"] * nk * D * 5 // 4
    if kind == "beams":
        groups, beams = _log(rng, 1, 8), rng.randint(2, 6)
        most = min(4000, 10 ** 9 // per_slot // (2 * groups))
        length = _log(rng, 20, max(20, most))
        return dict(kind=kind, groups=groups, beams=beams, length=length, tail=rng.randint(1, max(1, min(200, length // 4))),
                    **pool)
    if kind == "compact":
        n_seq = _log(rng, 1, 32)
        length = _log(rng, 16, max(16, min(16000, 5 * 10 ** 8 // per_slot // n_seq)))
        tail = rng.choice([min(length, rng.randint(1, 64)), rng.randint(length // 2, length)])
        return dict(kind=kind, n_seq=n_seq, length=length, tail=tail, kept=rng.choice([0.1, 0.5, 0.9]), **pool)
    n = _log(rng, 1, max(1, min(400, 8 * 10 ** 8 // per_slot // page)))
    return dict(kind=kind, n=n, n_page=n + rng.randint(0, 40), to_page=n + rng.randint(0, 60), **pool)


# ------------------------------------------------------------------ inputs

def _gen(seed, *more):
    g = torch.Generator(device="cuda")
    s = seed & 0xFFFFFFFF
    for m in more:
        s = (s * 1000003 + m + 1) & 0x7FFFFFFFFFFF
    g.manual_seed(s)
    return g


def _rng(seed, what):
    return np.random.default_rng([seed & 0x7FFFFFFF, what])


def _randn(g, shape):
    return torch.randn(shape, device="cuda", generator=g)


def _grid16(y, down):
    """float64 values rounded to half precision's (towards zero or to nearest even), still as float64."""
    _, e = torch.frexp(y)
    unit = ((torch.clamp_min(e.long() - 1, -14) - 10 + 1023) << 52).view(torch.float64)
    return (torch.trunc(y / unit) if down else torch.round(y / unit)) * unit


def _words16(step, low):
    """Half-precision values (as float64) as words: the step below, the lowest value above."""
    lo, st = low.to(torch.float16).view(torch.int16).int(), step.to(torch.float16).view(torch.int16).int()
    return (lo << 16) | (st & 0xFFFF)


def _quantise(x):
    """Rows [..., D] as codes (words of eight, [..., D / 8]) and steps with lowest values (words, [..., D / 32])."""
    g = x.unflatten(-1, (-1, 32)).double()
    mn, mx = g.amin(-1), g.amax(-1)
    bad = ~(g.abs().amax(-1) <= 65504.0)
    low = torch.where(bad, torch.zeros_like(mn), _grid16(torch.where(bad, torch.zeros_like(mn), mn), False))
    step = _grid16(torch.where(bad, torch.zeros_like(mn), (mx - low) / 15.0).clamp_min(0.0), True)
    live = step > 0
    code = torch.round((g - low[..., None]) / torch.where(live, step, torch.ones_like(step))[..., None])
    code = torch.where(live[..., None], code.clamp(0.0, 15.0), torch.zeros_like(code)).long()
    low = torch.where(bad, torch.full_like(low, math.nan), low)
    shifts = torch.tensor(SHIFTS, device=x.device)
    words = (code.unflatten(-1, (-1, 8)) << shifts).sum(-1).flatten(-2)
    return words.to(torch.int32), _words16(step, low)


def _split(pool, ps, D):
    """Views of a pool [..., words of a page's kv head]: key codes, value codes, key and value steps, each [..., ps, width]."""
    a, b = ps * D // 8, ps * D // 32
    return [pool[..., o:o + n * ps].unflatten(-1, (ps, n))
            for o, n in ((0, D // 8), (a, D // 8), (2 * a, D // 32), (2 * a + b, D // 32))]


def _values(words, meta):
    """Codes and their words of step and lowest value as the half-precision values they stand for (as float64)."""
    shifts = torch.tensor(SHIFTS, device=words.device)
    code = ((words[..., None] >> shifts) & 15).flatten(-2).unflatten(-1, (-1, 32)).double()
    step = (meta << 16 >> 16).to(torch.int16).view(torch.float16).double()
    low = (meta >> 16).to(torch.int16).view(torch.float16).double()
    return _grid16(low[..., None] + step[..., None] * code, False).flatten(-2)


def _pool_shape(c, n_layer, n_page):
    return (n_layer, n_page, c["n_head_kv"], c["page"] * c["head_dim"] * 5 // 16)


def _random_words(g, shape):
    return torch.randint(-2 ** 31, 2 ** 31, shape, dtype=torch.int32, device="cuda", generator=g)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _table(rng, lengths, ps, n_table, n_page):
    """Table rows of sequences of their own, their pages all over a pool."""
    need = [-(-int(n) // ps) for n in lengths]
    ids = rng.permutation(n_page).astype(np.int32)
    table, at = np.full((len(need), n_table), -1, np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    return table


def _refs(table, n_page):
    return np.bincount(table[table >= 0], minlength=n_page).astype(np.int32)


def _store_inputs(c, seed):
    """The projections [q | k | v] of new rows, of which k and v are stored."""
    rng, g = _rng(seed, 31), _gen(seed, 1)
    nh, nk, D = c["n_head"], c["n_head_kv"], c["head_dim"]
    n_table = -(-c["slots"] // c["page"])
    n_page = c["n_seq"] * n_table + 3
    table = _table(rng, [c["slots"]] * c["n_seq"], c["page"], n_table, n_page)
    start = rng.integers(0, c["slots"] - c["rows"] + 1, c["n_seq"]).astype(np.int32)
    qkv = _randn(g, (c["n_seq"] * c["rows"], nh + 2 * nk, D)) + 2.0 * _randn(g, (nh + 2 * nk, D))
    qkv = (qkv * torch.exp(0.5 * _randn(g, qkv.shape[:2]))[..., None]).to(TYPES[c["type"]])
    return dict(table=_cuda(table), refs=_cuda(_refs(table, n_page)), start=_cuda(start), qkv=qkv.flatten(1))


def _lengths(c, seed):
    """Per sequence: slots cached and rows of queries; which rows each sees, as truth values (None: those before it)."""
    rng = _rng(seed, 32)
    n, T, P = c["n_seq"], c["rows"], c["prefix"]
    prefix, count = np.full(n, P, np.int32), np.full(n, T, np.int32)
    if c["ragged"]:
        prefix = rng.integers(max(0, P - P // 4), P + 1, n).astype(np.int32)
        count = rng.integers(0, T + 1, n).astype(np.int32) if T > 1 else count
        count[rng.integers(0, n)] = T
    sees = None
    if c["tree"]:
        sees = np.zeros((n, T, T), bool)
        for s in range(n):
            for t in range(T):
                if t:
                    sees[s, t] = sees[s, t - 1 if rng.random() < 0.4 else int(rng.integers(0, t))]
                sees[s, t, t] = True
    return prefix, count, sees


def _mask_words(sees):
    """[n][T][T] truth values as [n][T][ceil(T / 64)] words of 64 bits."""
    n, T, _ = sees.shape
    bits = np.zeros((n, T, (T + 63) // 64 * 64), bool)
    bits[..., :T] = sees
    return np.packbits(bits, axis=-1, bitorder="little").view(np.int64)


def _attention_inputs(c, seed):
    """A layer whose slots hold keys with channels of their own means, and values; the other layer's and the spare pages
    hold anything."""
    g = _gen(seed, 2)
    n, nh, nk, D, ps = c["n_seq"], c["n_head"], c["n_head_kv"], c["head_dim"], c["page"]
    prefix, count, sees = _lengths(c, seed)
    n_table = -(-(c["prefix"] + c["rows"]) // ps) + 1
    n_page = n * n_table + 2
    table = _table(_rng(seed, 33), prefix + c["rows"], ps, n_table, n_page)
    pool = _random_words(g, _pool_shape(c, 2, n_page))
    mean = _randn(g, (nk, 1, D))
    for s in range(n):
        ids = _cuda(table[s][table[s] >= 0]).long()
        for i, parts in ((0, 1.0), (1, 0.0)):
            x = _randn(g, (len(ids), nk, ps, D)) + parts * mean
            x = x * torch.exp(0.3 * _randn(g, x.shape[:3]))[..., None]
            words, meta = _quantise(x)
            views = _split(pool[1], ps, D)
            views[i][ids], views[2 + i][ids] = words, meta
    q = (1.5 * _randn(g, (n * c["rows"], nh * D))).to(TYPES[c["type"]])
    return dict(pool=pool, table=table, refs=_refs(table, n_page), prefix=prefix, count=count, sees=sees, q=q)


def _beam_inputs(c, seed):
    """Groups of beams that share a prompt's pages and have tails of their own; each beam's parent among its group's."""
    rng = _rng(seed, 34)
    B, ps, n = c["beams"], c["page"], c["groups"] * c["beams"]
    length = np.repeat(rng.integers(c["length"] - c["length"] // 8, c["length"] + 1, c["groups"]), B).astype(np.int32)
    n_table = -(-(c["length"] + 1) // ps) + 1
    shared = np.maximum(length - c["tail"], 0) // ps  # whole pages of the prompt
    need = -(-length // ps)
    n_page = c["groups"] * (-(-c["length"] // ps)) + n * (-(-c["tail"] // ps) + 2) + 4
    ids, at = rng.permutation(n_page).astype(np.int32), 0
    table = np.full((n, n_table), -1, np.int32)
    for s in range(n):
        first = 0 if s % B == 0 else shared[s]
        table[s, :first] = table[s - s % B, :first]
        table[s, first:need[s]] = ids[at:at + need[s] - first]
        at += need[s] - first
    parent = (np.arange(n) // B * B + rng.integers(0, B, n)).astype(np.int32)
    return dict(pool=_random_words(_gen(seed, 3), _pool_shape(c, c["n_layer"], n_page)), table=_cuda(table),
                refs=_cuda(_refs(table, n_page)), parent=_cuda(parent), length=_cuda(length), want=_cuda(length + 1))


def _compact_inputs(c, seed):
    """Sequences of whose last slots some are kept."""
    rng = _rng(seed, 35)
    n, T, ps = c["n_seq"], c["tail"], c["page"]
    length = rng.integers(max(T, c["length"] - c["length"] // 8), c["length"] + 1, n).astype(np.int32)
    first = (length - T).astype(np.int32)
    most = max(1, int(T * c["kept"]))
    count = rng.integers(most // 2, most + 1, n).astype(np.int32)
    rows = np.zeros((n, most), np.int32)
    for s in range(n):
        rows[s, :count[s]] = first[s] + np.sort(rng.permutation(T)[:count[s]])
    n_page = n * (-(-c["length"] // ps)) + 5
    table = _table(rng, length, ps, -(-c["length"] // ps) + 1, n_page)
    return dict(pool=_random_words(_gen(seed, 4), _pool_shape(c, c["n_layer"], n_page)), table=_cuda(table),
                refs=_cuda(_refs(table, n_page)), first=_cuda(first), length=_cuda(length), rows=_cuda(rows),
                count=_cuda(count), keep=_cuda(first + count))


def _copy_inputs(c, seed):
    rng = _rng(seed, 36)
    return dict(pool=_random_words(_gen(seed, 5), _pool_shape(c, c["n_layer"], c["n_page"])),
                to=torch.zeros(_pool_shape(c, c["n_layer"], c["to_page"]), dtype=torch.int32, device="cuda"),
                src=_cuda(rng.permutation(c["n_page"])[:c["n"]].astype(np.int32)),
                dst=_cuda(rng.permutation(c["to_page"])[:c["n"]].astype(np.int32)))


def prepare(case, seed):
    c, kind = case, case["kind"]
    if kind == "store":
        s = _store_inputs(c, seed)
        s["pool"] = torch.zeros(_pool_shape(c, 2, s["refs"].numel()), dtype=torch.int32, device="cuda")
        s["slots"] = s["start"][:, None] + torch.arange(c["rows"], device="cuda", dtype=torch.int32)
        shape = (c["n_seq"] * c["rows"], c["n_head_kv"] * c["head_dim"])
        s["k_out"], s["v_out"] = (torch.zeros(shape, dtype=TYPES[c["type"]], device="cuda") for _ in range(2))
    elif kind == "attention":
        s = _attention_inputs(c, seed)
        s["out"] = torch.zeros_like(s["q"])
        s["max_prefix"] = int(s["prefix"].max())
        s["mask"] = None if s["sees"] is None else _cuda(_mask_words(s["sees"]))
        for n in ("table", "refs", "prefix", "count"):
            s[n] = _cuda(s[n])
    else:
        s = dict(beams=_beam_inputs, compact=_compact_inputs, copy=_copy_inputs)[kind](c, seed)
        s["missing"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    s["case"] = c
    if own:
        import kanjoos_amd as K

        K.open_device(0)
        s["stream"] = torch.cuda.current_stream().cuda_stream

        def pages(pool, table=None, refs=None):
            n_seq, n_table = (1, 1) if table is None else table.shape
            return K.KvPages(pool.shape[0], pool.shape[1], c["page"], c["n_head_kv"], c["head_dim"], n_seq, n_table,
                             pool.data_ptr(), None if table is None else table.data_ptr(),
                             None if refs is None else refs.data_ptr())

        if kind == "copy":
            s["pages"], s["to_pages"] = pages(s["pool"]), pages(s["to"])
        else:
            s["pages"] = pages(s["pool"], s["table"], s["refs"])
        if kind == "attention":
            s["workspace"] = K.DeviceBuffer(max(16, K.attention_pages_workspace(s["pages"], c["n_head"], c["rows"],
                                                                               s["max_prefix"])))
        if kind in ("beams", "compact"):
            s["workspace"] = K.DeviceBuffer(K.pages_workspace(s["pages"]))
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ one pass through the framework

def _run_own(s, c):
    import kanjoos_amd as K

    kind, stream, pages = c["kind"], s["stream"], s["pages"]
    if kind == "store":
        nh, nk, D = c["n_head"], c["n_head_kv"], c["head_dim"]
        typ, size = TYPE_IDS[c["type"]], s["qkv"].element_size()
        k = s["qkv"].data_ptr() + nh * D * size
        K.pages_store(pages, 1, typ, k, k + nk * D * size, s["start"].data_ptr(), c["rows"], row_stride=(nh + 2 * nk) * D,
                      stream=stream)
        K.pages_load(pages, 1, typ, s["k_out"].data_ptr(), s["v_out"].data_ptr(), c["rows"], slots=s["slots"].data_ptr(),
                     stream=stream)
        return s["k_out"], s["v_out"]
    if kind == "attention":
        K.attention_pages(pages, 1, TYPE_IDS[c["type"]], s["q"].data_ptr(), s["out"].data_ptr(), c["n_head"], c["rows"],
                          s["prefix"].data_ptr(), s["max_prefix"], s["workspace"], counts=s["count"].data_ptr(),
                          mask=None if s["mask"] is None else s["mask"].data_ptr(), stream=stream)
        return s["out"]
    if kind == "beams":
        K.pages_fork(pages, s["parent"].data_ptr(), s["workspace"], keep=s["length"].data_ptr(), stream=stream)
        K.pages_reserve(pages, s["length"].data_ptr(), s["want"].data_ptr(), s["missing"].data_ptr(), s["workspace"],
                        stream=stream)
    elif kind == "compact":
        K.pages_reserve(pages, s["length"].data_ptr(), s["length"].data_ptr(), s["missing"].data_ptr(), s["workspace"],
                        start=s["first"].data_ptr(), stream=stream)
        K.pages_compact(pages, s["first"].data_ptr(), s["rows"].data_ptr(), s["rows"].shape[1], counts=s["count"].data_ptr(),
                        stream=stream)
        K.pages_free(pages, s["keep"].data_ptr(), stream=stream)
    else:
        K.pages_copy(s["to_pages"], pages, s["dst"].data_ptr(), s["src"].data_ptr(), c["n"], stream=stream)
        return s["to"]
    return {n: s[n] for n in ("table", "refs", "missing", "pool")}


# ------------------------------------------------------------------ one pass in plain torch

def _place(s, c, seq, slot):
    """Page and row of slots of sequences."""
    return s["table"].long()[seq, slot // c["page"]], slot % c["page"]


def _seen(s, c, L):
    """[n_seq][rows][L]: the slots each row attends to."""
    T = c["rows"]
    slot, bit = torch.arange(L, device="cuda"), torch.arange(T, device="cuda")
    u = slot[None] - s["prefix"][:, None].long()  # [n_seq][L]: the row in a slot
    if s["mask"] is None:
        rows = u[:, None] <= bit[None, :, None]
    else:
        bits = (s["mask"][:, :, bit // 64] >> (bit % 64)) & 1  # [n_seq][T][T]
        rows = torch.gather(bits, 2, u.clamp(0, T - 1)[:, None, :].expand(-1, T, -1)).bool()
    inside = (u >= 0) & (u < s["count"][:, None])
    return (u < 0)[:, None] | (rows & inside[:, None])


def _attention_plain(s, c):
    n, nh, nk, D, T, ps = c["n_seq"], c["n_head"], c["n_head_kv"], c["head_dim"], c["rows"], c["page"]
    G, L = nh // nk, s["max_prefix"] + T
    entries = -(-L // ps)
    page = s["table"][:, :entries].long().clamp_min(0)
    kc, vc, km, vm = _split(s["pool"][1], ps, D)

    def rows(words, meta):  # [n_seq][nk][L][D]
        x = _values(words[page], meta[page]).float()
        return x.permute(0, 2, 1, 3, 4).reshape(n, nk, entries * ps, D)[:, :, :L]

    kk, vv = rows(kc, km), rows(vc, vm)
    q = s["q"].view(n, T, nk, G, D).permute(0, 2, 1, 3, 4).reshape(n, nk, T * G, D).float()
    seen = _seen(s, c, L)
    vv = vv.masked_fill(~seen.any(1)[:, None, :, None], 0.0)  # (slots behind a sequence hold anything)
    kk = kk.masked_fill(~seen.any(1)[:, None, :, None], 0.0)
    scores = torch.matmul(q, kk.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
    seen = seen[:, None, :, None].expand(n, nk, T, G, L).reshape(n, nk, T * G, L)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, vv) / torch.where(total == 0, torch.ones_like(total), total)
    o = o.view(n, nk, T, G, D).permute(0, 2, 1, 3, 4).reshape(n, T, nh * D)
    live = torch.arange(T, device="cuda")[None] < s["count"][:, None]
    return torch.where(live[..., None], o, torch.zeros_like(o)).to(TYPES[c["type"]]).view(n * T, nh * D)


def _fork_plain(s, c, parent, keep):
    table, refs = s["table"], s["refs"]
    n, n_table = table.shape
    entry = torch.arange(n_table, device="cuda")
    new = torch.where(entry[None] * c["page"] < keep[:, None], table[parent.long()], torch.full_like(table, -1))
    for t, sign in ((new, 1), (table, -1)):
        refs.scatter_add_(0, t.clamp_min(0).long().view(-1), sign * (t >= 0).int().view(-1))
    table.copy_(new)


def _reserve_plain(s, c, start, length, want):
    table, refs, ps = s["table"], s["refs"], c["page"]
    n, n_table = table.shape
    n_page = refs.numel()
    entry = torch.arange(n_table, device="cuda")[None]
    flat = torch.arange(n * n_table, device="cuda").view(n, n_table)
    need = (entry * ps < want[:, None]) & ((entry + 1) * ps > start[:, None])
    held, at = table >= 0, table.clamp_min(0).long()
    shared = need & held & (refs[at] > 1)
    # a page that all its holders write stays with the last of them
    asked = torch.zeros_like(refs).scatter_add_(0, at.view(-1), shared.int().view(-1))
    last = torch.full((n_page,), -1, device="cuda").scatter_reduce_(
        0, at.view(-1), torch.where(shared, flat, torch.full_like(flat, -1)).view(-1), "amax")
    fresh = need & (~held | (shared & ~((asked[at] == refs[at]) & (last[at] == flat))))
    unused = refs <= 0
    order = torch.argsort((~unused).int(), stable=True)
    rank = (torch.cumsum(fresh.view(-1).int(), 0) - 1).clamp(0, n_page - 1).view(n, n_table)
    short = (fresh.sum() - unused.sum()).clamp_min(0)
    fresh = fresh & (short == 0)
    new = torch.where(fresh, order[rank].int(), table)
    seq, ent = fresh.nonzero(as_tuple=True)
    src, dst = at[seq, ent], new[seq, ent].long()
    rows = torch.where(held[seq, ent], (length[seq] - ent * ps).clamp(0, ps), torch.zeros_like(ent))
    kept = (torch.arange(ps, device="cuda")[None] < rows[:, None])[None, :, None, :, None]
    for part in _split(s["pool"], ps, c["head_dim"]):
        part[:, dst] = torch.where(kept, part[:, src], part[:, dst])
    refs.scatter_add_(0, at[seq, ent], -held[seq, ent].int())
    refs[dst] = 1
    table.copy_(new)
    s["missing"].copy_(short)


def _compact_plain(s, c):
    ps, n_rows = c["page"], s["rows"].shape[1]
    seq, i = (torch.arange(n_rows, device="cuda")[None] < s["count"][:, None]).nonzero(as_tuple=True)
    src_page, src_row = _place(s, c, seq, s["rows"].long()[seq, i])
    dst_page, dst_row = _place(s, c, seq, s["first"].long()[seq] + i)
    for part in _split(s["pool"], ps, c["head_dim"]):
        part[:, dst_page, :, dst_row] = part[:, src_page, :, src_row]


def _free_plain(s, c, keep):
    table, refs = s["table"], s["refs"]
    entry = torch.arange(table.shape[1], device="cuda")
    gone = (entry[None] * c["page"] >= keep[:, None]) & (table >= 0)
    refs.scatter_add_(0, table.clamp_min(0).long().view(-1), -gone.int().view(-1))
    table.masked_fill_(gone, -1)


def _run_plain(s, c):
    kind = c["kind"]
    if kind == "store":
        n, nh, nk, D, T = c["n_seq"], c["n_head"], c["n_head_kv"], c["head_dim"], c["rows"]
        page, row = _place(s, c, torch.arange(n, device="cuda")[:, None], s["slots"].long())
        x = s["qkv"].view(n, T, nh + 2 * nk, D)
        parts = _split(s["pool"][1], c["page"], D)
        out = []
        for i in range(2):
            words, meta = _quantise(x[:, :, nh + i * nk:nh + (i + 1) * nk].float())
            parts[i][page, :, row], parts[2 + i][page, :, row] = words, meta
            out.append(_values(parts[i][page, :, row], parts[2 + i][page, :, row]).to(TYPES[c["type"]]).reshape(n * T, nk * D))
        return tuple(out)
    if kind == "attention":
        return _attention_plain(s, c)
    if kind == "beams":
        _fork_plain(s, c, s["parent"], s["length"])
        _reserve_plain(s, c, s["length"], s["length"], s["want"])
    elif kind == "compact":
        _reserve_plain(s, c, s["first"], s["length"], s["length"])
        _compact_plain(s, c)
        _free_plain(s, c, s["keep"])
    else:
        s["to"][:, s["dst"].long()] = s["pool"][:, s["src"].long()]
        return s["to"]
    return {n: s[n] for n in ("table", "refs", "missing", "pool")}


def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c, kind = case, case["kind"]
    nk, D = c["n_head_kv"], c["head_dim"]
    slot = 1.25 * nk * D  # bytes of a slot's keys and values in one layer: each half a byte and an eighth a dim
    size = 4 if c.get("type") == "f32" else 2
    if kind == "store":
        rows = c["n_seq"] * c["rows"]
        return dict(bytes=rows * (2 * slot + 4 * nk * D * size + 8), flops=10.0 * rows * 2 * nk * D)
    if kind == "attention":
        # (of a ragged batch: the sequences' mean prefix and rows)
        prefix = c["prefix"] * (0.875 if c["ragged"] else 1.0)
        rows = c["rows"] * (0.5 if c["ragged"] and c["rows"] > 1 else 1.0)
        return dict(bytes=c["n_seq"] * ((prefix + rows) * slot + rows * 2 * c["n_head"] * D * size),
                    flops=4.0 * c["n_seq"] * rows * c["n_head"] * D * (prefix + rows / 2))
    slot *= c["n_layer"]
    if kind == "beams":
        n = c["groups"] * c["beams"]
        held = -(-c["length"] // c["page"])
        # of the parents' last pages all holders but one get a copy, of half a page on average; about e^-1 have no child
        return dict(bytes=n * 0.37 * slot * c["page"] + 16 * n * held, flops=1.0 * n * held)
    if kind == "compact":
        rows = 0.75 * max(1, int(c["tail"] * c["kept"])) * c["n_seq"]
        return dict(bytes=rows * 2 * slot, flops=rows)
    return dict(bytes=2.0 * c["n"] * c["page"] * slot, flops=1.0 * c["n"])


# ------------------------------------------------------------------ the definitions in 64 bits

def _half64(x):
    """Half precision by numpy's own conversion from float64."""
    with np.errstate(over="ignore"):
        return x.astype(np.float16).astype(np.float64)


def _decode64(codes, meta):
    """One matrix's words as float64 values."""
    codes, meta = (np.ascontiguousarray(t.cpu().numpy()).view(np.uint32) for t in (codes, meta))
    half = meta.view(np.uint16).reshape(*meta.shape, 2).view(np.float16).astype(np.float64)
    nib = np.stack([(codes >> s) & 15 for s in SHIFTS], -1).reshape(*codes.shape[:-1], -1, 32)
    return _half64(half[..., 1:] + half[..., :1] * nib).reshape(*codes.shape[:-1], -1)


def _store64(x):
    """Rows [..., D] as the cache holds them, group by group of 32."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    low = _half64(g.min(-1))
    room = np.maximum(g.max(-1) - low, 0.0) / 15.0
    step = _half64(room)
    step = np.where(step > room, np.nextafter(step.astype(np.float16), np.float16(0)).astype(np.float64), step)
    code = np.clip(np.rint((g - low[..., None]) / np.where(step > 0, step, np.inf)[..., None]), 0, 15)
    return _half64(low[..., None] + step[..., None] * code).reshape(x.shape)


def _attention64(c, seed):
    s = _attention_inputs(c, seed)
    n, nh, nk, D, T, ps = c["n_seq"], c["n_head"], c["n_head_kv"], c["head_dim"], c["rows"], c["page"]
    G = nh // nk
    q = s["q"].double().view(n, T, nk, G, D)
    out = torch.zeros((n, T, nk, G, D), dtype=torch.float64, device="cuda")
    a, b = ps * D // 8, ps * D // 32
    for i in range(n):
        P, N = int(s["prefix"][i]), int(s["count"][i])
        if N == 0:
            continue
        ids = _cuda(s["table"][i][:-(-(P + N) // ps)]).long()
        words = s["pool"][1][ids].transpose(0, 1)  # [nk][pages][words]
        sees = np.tril(np.ones((N, N), bool)) if s["sees"] is None else s["sees"][i, :N, :N]
        hidden = torch.from_numpy(~sees).cuda()
        for h in range(nk):
            w = words[h].contiguous()
            kk, vv = (_cuda(_decode64(w[:, o:o + a].reshape(-1, D // 8), w[:, m:m + b].reshape(-1, D // 32))[:P + N])
                      for o, m in ((0, 2 * a), (a, 2 * a + b)))
            for j in range(G):
                x = q[i, :N, h, j] @ kk.T.contiguous() / math.sqrt(D)
                x[:, P:].masked_fill_(hidden, -math.inf)
                out[i, :N, h, j] = torch.softmax(x, -1) @ vv
    return out.view(n * T, nh * D)


def _tables64(c, table, refs, steps):
    """The table's steps entry by entry, in order, on the host: ("fork", parent, keep), ("reserve", start, length, want),
    ("free", keep).  Returns the pages that reserving copies as (source, destination, rows)."""
    ps, copies = c["page"], []
    n, n_table = table.shape
    for step, *args in steps:
        if step == "fork":
            old = table.copy()
            for s in range(n):
                for e in range(n_table):
                    table[s, e] = old[args[0][s], e] if e * ps < args[1][s] else -1
            refs[:] = _refs(table, len(refs))
        elif step == "reserve":
            start, length, want = args
            asked = [(s, e) for s in range(n) for e in range(start[s] // ps, n_table) if e * ps < want[s]]
            before = refs.copy()
            wanting = {}
            for s, e in asked:
                if table[s, e] >= 0 and before[table[s, e]] > 1:
                    wanting.setdefault(int(table[s, e]), []).append((s, e))
            stays = {v[-1] for p, v in wanting.items() if len(v) == before[p]}
            unused = iter(np.flatnonzero(before <= 0))
            for s, e in asked:
                p = int(table[s, e])
                if p >= 0 and (before[p] <= 1 or (s, e) in stays):
                    continue
                new = int(next(unused))
                if p >= 0:
                    refs[p] -= 1
                    copies.append((p, new, int(np.clip(length[s] - e * ps, 0, ps))))
                table[s, e], refs[new] = new, 1
        else:
            for s in range(n):
                for e in range(-(-int(args[0][s]) // ps), n_table):
                    if table[s, e] >= 0:
                        refs[table[s, e]] -= 1
                        table[s, e] = -1
    return copies


def _bytes_of(c, pool):
    """The pool as [layer][page][kv head] rows of bytes: four blocks of slots each."""
    ps, D = c["page"], c["head_dim"]
    raw = pool.view(torch.uint8)
    at, blocks = 0, []
    for width in (D // 2, D // 2, D // 8, D // 8):
        blocks.append(raw[..., at:at + ps * width].unflatten(-1, (ps, width)))
        at += ps * width
    return blocks


def exact(case, seed):
    c, kind = case, case["kind"]
    if kind == "store":
        s = _store_inputs(c, seed)
        nh, nk, D = c["n_head"], c["n_head_kv"], c["head_dim"]
        x = s["qkv"].view(-1, nh + 2 * nk, D).double().cpu().numpy()
        return tuple(_cuda(_store64(x[:, a:a + nk]).reshape(len(x), -1)) for a in (nh, nh + nk))
    if kind == "attention":
        return _attention64(c, seed)
    if kind == "copy":
        s = _copy_inputs(c, seed)
        for i, j in zip(s["src"].tolist(), s["dst"].tolist()):
            s["to"][:, j] = s["pool"][:, i]
        return s["to"]
    s = (_beam_inputs if kind == "beams" else _compact_inputs)(c, seed)
    h = {n: t.cpu().numpy() for n, t in s.items() if n != "pool"}
    table, refs = h["table"], h["refs"]
    blocks = _bytes_of(c, s["pool"])

    def copy(copies):
        for p, q, rows in copies:
            for b in blocks:
                b[:, q, :, :rows] = b[:, p, :, :rows]

    if kind == "beams":
        copy(_tables64(c, table, refs, [("fork", h["parent"], h["length"]), ("reserve", h["length"], h["length"], h["want"])]))
    else:
        copy(_tables64(c, table, refs, [("reserve", h["first"], h["length"], h["length"])]))
        for i in range(c["n_seq"]):
            m = int(h["count"][i])
            to, fro = h["first"][i] + np.arange(m), h["rows"][i, :m]
            put = [_cuda(x.astype(np.int64)) for x in (table[i, fro // c["page"]], fro % c["page"],
                                                       table[i, to // c["page"]], to % c["page"])]
            for b in blocks:
                b[:, put[2], :, put[3]] = b[:, put[0], :, put[1]].clone()
        _tables64(c, table, refs, [("free", h["keep"])])
    return dict(table=_cuda(table), refs=_cuda(refs), missing=torch.zeros(1, dtype=torch.int32), pool=s["pool"])
