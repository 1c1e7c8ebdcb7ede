"""Performance cases of the operators around a speculative decoding step.

One step drafts a tree of tokens, rotates the drafts' queries and keys at their
own positions (``rope``), writes their keys and values into the cache in its
format (``kv_store``; ``kv_load`` reads rows back), attends from every draft to
the cache and to its ancestors (``attention_tree``) and takes the drafts' log
probabilities from the logits (``token_logprobs``).

Kinds: ``rope``, ``kv`` (rows stored, then read back), ``load`` (rows gathered
from a cache), ``tree`` (attention) and ``logprobs``.  With ``own`` false,
``run`` computes a pass in elementary torch operations; with ``own`` true it
calls ``kanjoos_amd``.  ``exact`` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE_IDS = {"f32": 0, "f16": 1, "bf16": 30}
TINY = 2.0 ** -119  # rows of an 8-bit cache whose largest magnitude is below this are stored as zeros
A3B = dict(n_head=32, n_head_kv=4, head_dim=128)
HEADS = [(32, 4, 128), (32, 4, 128), (32, 8, 128), (16, 4, 128), (12, 4, 128), (8, 8, 64), (8, 2, 64), (16, 2, 64)]
PLAIN_ROPE = dict(layout="half", n_rot=128, norm=True, scaling="none", factor=1.0)


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one decode token's queries and keys, normalised and rotated: the smallest launch
        dict(name="rope_step", kind="rope", type="f32", rows=1, pos=4100, **PLAIN_ROPE, **A3B),
        # a long prompt far into a context stretched by YaRN
        dict(name="rope_prompt_yarn", kind="rope", type="f32", rows=4000, pos=90000,
             **dict(PLAIN_ROPE, scaling="yarn", factor=4.0), **A3B),
        # 32 sequences' new keys and values as int8, read back for the accepted rows
        dict(name="kv_step_i8", kind="kv", format="i8", type="f32", n_seq=32, rows=1, n_ctx=2304, **A3B),
        # a prompt's keys and values as e4m3
        dict(name="kv_prompt_f8", kind="kv", format="f8", type="f32", n_seq=1, rows=4096, n_ctx=4352, **A3B),
        # the accepted paths of 32 sequences gathered from among their drafts
        dict(name="load_paths_f8", kind="load", format="f8", type="f32", n_seq=32, rows=7, n_ctx=2304, **A3B),
        # a whole int8 prefix read back in half precision
        dict(name="load_prefix_i8", kind="load", format="i8", type="f16", n_seq=1, rows=32000, n_ctx=32768, **A3B),
        # a chain of four drafts at a short context, as the framework's own cache holds it: latency
        dict(name="tree_4_f16_1k", kind="tree", format="f16", type="f32", n_seq=1, drafts=4, prefix=1000, ragged=False,
             chain=True, **A3B),
        # an ordinary tree at a 4K context over an int8 cache
        dict(name="tree_25_i8_4k", kind="tree", format="i8", type="f32", n_seq=1, drafts=25, prefix=4100, ragged=False,
             chain=False, **A3B),
        # 32 sequences at about 2K each, up to 8 drafts a sequence, ragged
        dict(name="tree_32x8_f8_2k", kind="tree", format="f8", type="bf16", n_seq=32, drafts=8, prefix=2048, ragged=True,
             chain=False, **A3B),
        # a wide tree at the longest context: the largest
        dict(name="tree_64_f16_32k", kind="tree", format="f16", type="f16", n_seq=1, drafts=64, prefix=32700,
             ragged=False, chain=False, **A3B),
        # one step's token with the alternatives an answer lists
        dict(name="logprobs_step", kind="logprobs", type="f32", rows=1, vocab=151936, stride=151936, top=20,
             temperature=1.0),
        # a prompt's tokens scored
        dict(name="logprobs_prompt", kind="logprobs", type="f32", rows=500, vocab=151936, stride=151936, top=5,
             temperature=0.8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "kv", "load", "tree", "tree", "tree", "logprobs"])
    nh, nk, D = rng.choice(HEADS)
    heads = dict(n_head=nh, n_head_kv=nk, head_dim=D)
    typ = rng.choice(["f32", "f32", "f16", "bf16"])
    if kind == "rope":
        scaling = rng.choice(["none", "linear", "ntk", "yarn", "llama3"])
        return dict(kind=kind, type=typ, rows=_log(rng, 1, 4000), pos=_log(rng, 1, 200000),
                    layout=rng.choice(["half", "interleaved"]), n_rot=rng.choice([D, 8 * rng.randint(1, D // 8)]),
                    norm=rng.random() < 0.5, scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]), **heads)
    form = rng.choice(["f16", "f8", "i8"])
    if kind == "kv":
        n_seq = _log(rng, 1, 32)
        rows = _log(rng, 1, 4096 // n_seq)
        return dict(kind=kind, format=form, type=typ, n_seq=n_seq, rows=rows, n_ctx=rows + rng.randint(1, 300), **heads)
    if kind == "load":
        n_seq = _log(rng, 1, 32)
        rows = _log(rng, 1, 32000 // n_seq)
        return dict(kind=kind, format=form, type=typ, n_seq=n_seq, rows=rows, n_ctx=rows + rng.randint(0, 800), **heads)
    if kind == "tree":
        n_seq = rng.choice([1, 1, _log(rng, 2, 32)])
        drafts = _log(rng, 1, 64)
        # no more work than the largest listed case, and no more cache than the batched one's fourfold
        most = min(32700, 64 * 32 * 32700 // (n_seq * drafts * nh), 4 * 32 * 2048 // n_seq)
        return dict(kind=kind, format=form, type=typ, n_seq=n_seq, drafts=drafts, prefix=_log(rng, 1, most),
                    ragged=rng.random() < 0.5, chain=rng.random() < 0.3, **heads)
    vocab = _log(rng, 1000, 151936)
    return dict(kind=kind, type=typ, rows=_log(rng, 1, 500), vocab=vocab, stride=vocab + rng.choice([0, 0, 1, 64]),
                top=rng.choice([0, 1, 5, 20]), temperature=rng.choice([1.0, 1.0, 0.7, 1.3]))


# ------------------------------------------------------------------ inputs

def _gen(seed, *more):
    g = torch.Generator(device="cuda")
    s = seed & 0xFFFFFFFF
    for m in more:
        s = (s * 1000003 + m + 1) & 0x7FFFFFFFFFFF
    g.manual_seed(s)
    return g


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def _inv_freq64(c):
    """Rotation frequencies in float64 (numpy) and the factor of cos and sin, from the published scalings."""
    n, base, f, orig = c["n_rot"], 1e6, c["factor"], 32768
    if c["scaling"] == "ntk":
        base = base * f ** (n / (n - 2.0)) if n > 2 else base * f
    inv = base ** (-2.0 * np.arange(n // 2) / n)
    if c["scaling"] == "linear":
        return inv / f, 1.0
    if c["scaling"] == "yarn":
        def dim(turns):
            return n * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(dim(32.0)), 0), min(math.ceil(dim(1.0)), n - 1)
        ramp = np.clip((np.arange(n // 2) - lo) / (hi - lo if hi > lo else 0.001), 0, 1)
        return inv / f * ramp + inv * (1 - ramp), 0.1 * math.log(f) + 1.0
    if c["scaling"] == "llama3":
        wave = 2 * math.pi / inv
        smooth = np.clip((orig / wave - 1.0) / (4.0 - 1.0), 0, 1)
        return (1 - smooth) * inv / f + smooth * inv, 1.0
    return inv, 1.0


def _quantise(x, form):
    """Rows x [..., D] (float32) in the cache's format: codes and, for 8 bits, a scale a row.  The code is the exact
    quotient's (ties to even), so the quotients are taken in float64."""
    if form == "f16":
        return x.to(torch.float16), None
    top = 127.0 if form == "i8" else 448.0
    amax = x.abs().amax(-1)
    live = amax >= TINY
    y = x.double() * top / torch.where(live, amax, torch.full_like(amax, math.inf)).double()[..., None]
    if form == "i8":
        code = torch.round(y).to(torch.int8)
    else:  # three bits after the leading one, steps of 2^-9 below 2^-6
        step = torch.ldexp(torch.ones_like(y), torch.frexp(y).exponent.clamp_min(-5) - 4)
        code = (torch.round(y / step) * step).float().to(torch.float8_e4m3fn)
    return code, torch.where(live, amax / top, torch.zeros_like(amax))


def _values(code, scale):
    return code.float() if scale is None else code.float() * scale[..., None]


def _empty_cache(c):
    shape = (c["n_seq"], c["n_head_kv"], c["n_ctx"], c["head_dim"])
    dt = dict(f16=torch.float16, f8=torch.float8_e4m3fn, i8=torch.int8)[c["format"]]
    s = dict(k=torch.zeros(shape, dtype=dt, device="cuda"), v=torch.zeros(shape, dtype=dt, device="cuda"),
             k_scale=None, v_scale=None)
    if c["format"] != "f16":
        s["k_scale"], s["v_scale"] = (torch.zeros(shape[:3], device="cuda") for _ in range(2))
    return s


def _filled_cache(c, seed):
    """A cache whose every slot holds a key and a value; keys' and values' sizes vary from slot to slot."""
    s = _empty_cache(c)
    for i in range(c["n_seq"]):
        g = _gen(seed, 20, i)
        for n in ("k", "v"):
            x = _randn(g, s[n].shape[1:]) * torch.exp(0.3 * _randn(g, s[n].shape[1:3]))[..., None]
            code, scale = _quantise(x, c["format"])
            s[n][i] = code
            if scale is not None:
                s[n + "_scale"][i] = scale
    return s


def _tree(c, seed):
    """Per sequence: cached slots, drafts, and the drafts each draft sees (its ancestors and itself) as truth values."""
    rng = np.random.default_rng([seed & 0x7FFFFFFF, 21])
    n, T, P = c["n_seq"], c["drafts"], c["prefix"]
    prefix, count = np.full(n, P, np.int32), np.full(n, T, np.int32)
    if c["ragged"]:
        prefix = rng.integers(max(0, P - P // 4), P + 1, n).astype(np.int32)
        count = rng.integers(0, T + 1, n).astype(np.int32)
        count[rng.integers(0, n)] = T
    sees = np.zeros((n, T, T), bool)
    for s in range(n):
        for t in range(T):
            if t:
                parent = t - 1 if c["chain"] or rng.random() < 0.4 else int(rng.integers(0, t))
                sees[s, t] = sees[s, parent]
            sees[s, t, t] = True
    return prefix, count, sees


def _words(sees):
    """[n][T][T] truth values as [n][T][ceil(T/64)] words of 64 bits."""
    n, T, _ = sees.shape
    bits = np.zeros((n, T, (T + 63) // 64 * 64), bool)
    bits[..., :T] = sees
    return np.packbits(bits, axis=-1, bitorder="little").view(np.int64)


def _rope_inputs(c, seed):
    g = _gen(seed, 1)
    nh, nk, D, n = c["n_head"], c["n_head_kv"], c["head_dim"], c["rows"]
    qkv = _randn(g, (n, nh + 2 * nk, D), TYPES[c["type"]]).reshape(n, -1)
    inv, mscale = _inv_freq64(c)
    w = [1.0 + 0.1 * _randn(g, (D,)) for _ in range(2)]
    return dict(qkv=qkv, inv=torch.from_numpy(inv).cuda(), mscale=mscale, q_norm=w[0] if c["norm"] else None,
                k_norm=w[1] if c["norm"] else None,
                pos=(c["pos"] + torch.arange(n, device="cuda")).to(torch.int32))


def _kv_inputs(c, seed):
    """The projections [q | k | v] of new rows, of which k and v are stored."""
    g = _gen(seed, 2)
    nh, nk, D = c["n_head"], c["n_head_kv"], c["head_dim"]
    qkv = _randn(g, (c["n_seq"] * c["rows"], nh + 2 * nk, D))
    qkv = (qkv * torch.exp(0.5 * _randn(g, qkv.shape[:2]))[..., None]).to(TYPES[c["type"]])
    room = c["n_ctx"] - c["rows"] + 1
    start = torch.randint(0, room, (c["n_seq"],), device="cuda", generator=g).to(torch.int32)
    return dict(qkv=qkv.reshape(qkv.shape[0], -1), start=start)


def _load_slots(c, seed):
    rng = np.random.default_rng([seed & 0x7FFFFFFF, 22])
    return np.stack([np.sort(rng.permutation(c["n_ctx"])[:c["rows"]]) for _ in range(c["n_seq"])]).astype(np.int32)


def _logit_inputs(c, seed):
    """Logits with a few likely tokens; in every fourth row most of the vocabulary is ruled out."""
    g = _gen(seed, 3)
    n, V = c["rows"], c["vocab"]
    x = torch.full((n, c["stride"]), 50.0, dtype=TYPES[c["type"]], device="cuda")  # columns past the vocabulary
    for i in range(0, n, 64):
        m = min(64, n - i)
        y = 2.5 * _randn(g, (m, V))
        likely = torch.randint(0, V, (m, 12), device="cuda", generator=g)
        y.scatter_add_(1, likely, 8.0 + 3.0 * _randn(g, (m, 12)))
        ruled = torch.rand((m, V), device="cuda", generator=g) < 0.9
        ruled &= (torch.arange(i, i + m, device="cuda") % 4 == 3)[:, None]
        y = y.masked_fill(ruled, -math.inf)
        x[i:i + m, :V] = y.to(x.dtype)
    tokens = torch.randint(0, V, (n,), device="cuda", generator=g).to(torch.int32)
    for i in (0, 3):  # a greedy draft, and a row under a grammar (whose token is one of the allowed)
        tokens[i::4] = x[i::4, :V].argmax(-1).to(torch.int32)
    return dict(x=x, tokens=tokens)


def prepare(case, seed):
    c, kind = case, case["kind"]
    if kind == "rope":
        s = _rope_inputs(c, seed)
        nh, nk, D = c["n_head"], c["n_head_kv"], c["head_dim"]
        s["q_out"] = torch.empty((c["rows"], nh * D), dtype=TYPES[c["type"]], device="cuda")
        s["k_out"] = torch.empty((c["rows"], nk * D), dtype=TYPES[c["type"]], device="cuda")
    elif kind == "kv":
        s = _kv_inputs(c, seed)
        s.update(_empty_cache(c))
        s["slots"] = s["start"][:, None] + torch.arange(c["rows"], device="cuda", dtype=torch.int32)
        shape = (c["n_seq"] * c["rows"], c["n_head_kv"] * c["head_dim"])
        s["k_out"], s["v_out"] = (torch.zeros(shape, dtype=TYPES[c["type"]], device="cuda") for _ in range(2))
    elif kind == "load":
        s = _filled_cache(c, seed)
        s["slots"] = torch.from_numpy(_load_slots(c, seed)).cuda()
        shape = (c["n_seq"] * c["rows"], c["n_head_kv"] * c["head_dim"])
        s["k_out"], s["v_out"] = (torch.zeros(shape, dtype=TYPES[c["type"]], device="cuda") for _ in range(2))
    elif kind == "tree":
        c = dict(c, n_ctx=c["prefix"] + c["drafts"] + 33)
        prefix, count, sees = _tree(c, seed)
        s = _filled_cache(c, seed)
        g = _gen(seed, 4)
        shape = (c["n_seq"] * c["drafts"], c["n_head"] * c["head_dim"])
        s["q"] = (1.5 * _randn(g, shape)).to(TYPES[c["type"]])
        s["out"] = torch.zeros(shape, dtype=TYPES[c["type"]], device="cuda")
        s["prefix"], s["count"] = torch.from_numpy(prefix).cuda(), torch.from_numpy(count).cuda()
        s["max_prefix"] = int(prefix.max())
        s["mask"] = torch.from_numpy(_words(sees)).cuda()
    else:
        s = _logit_inputs(c, seed)
        n, top = c["rows"], c["top"]
        s["logprob"], s["entropy"] = (torch.empty(n, device="cuda") for _ in range(2))
        s["top_idx"] = torch.empty((n, top), dtype=torch.int32, device="cuda")
        s["top_logprob"] = torch.empty((n, top), device="cuda")
    s["case"] = c
    if own:
        import kanjoos_amd as K

        K.open_device(0)
        s["stream"] = torch.cuda.current_stream().cuda_stream
        if kind in ("kv", "load", "tree"):
            form = dict(f16=K.KV_F16, f8=K.KV_F8, i8=K.KV_I8)[c["format"]]
            s["cache"] = K.KvCache(form, c["n_seq"], c["n_head_kv"], c["n_ctx"], c["head_dim"], _p(s["k"]), _p(s["v"]),
                                   _p(s["k_scale"]), _p(s["v_scale"]))
        if kind == "tree":
            s["workspace"] = K.DeviceBuffer(K.attention_tree_workspace(s["cache"], c["n_head"], c["drafts"],
                                                                      s["max_prefix"]))
        if kind == "logprobs":
            s["workspace"] = K.DeviceBuffer(K.token_logprobs_workspace(c["rows"], c["vocab"]))
    torch.cuda.synchronize()
    return s


# ------------------------------------------------------------------ one pass through the framework

def _p(t):
    return None if t is None else t.data_ptr()


def _run_own(s, c):
    import kanjoos_amd as K

    kind, typ, stream = c["kind"], TYPE_IDS[c["type"]], s["stream"]
    if kind == "rope":
        nh, nk, D = c["n_head"], c["n_head_kv"], c["head_dim"]
        row = (nh + 2 * nk) * D
        q = s["qkv"].data_ptr()
        K.rope(typ, q, q + nh * D * s["qkv"].element_size(), s["pos"].data_ptr(), s["inv"].data_ptr(), c["rows"], nh, nk, D,
               s["q_out"].data_ptr(), s["k_out"].data_ptr(), n_rot=c["n_rot"],
               layout=K.ROPE_HALF if c["layout"] == "half" else K.ROPE_INTERLEAVED, mscale=s["mscale"],
               q_norm=_p(s["q_norm"]), k_norm=_p(s["k_norm"]), eps=EPS, q_stride=row, k_stride=row, stream=stream)
        return s["q_out"], s["k_out"]
    if kind == "kv":
        nh, nk, D = c["n_head"], c["n_head_kv"], c["head_dim"]
        size = s["qkv"].element_size()
        k = s["qkv"].data_ptr() + nh * D * size
        K.kv_store(s["cache"], typ, k, k + nk * D * size, s["start"].data_ptr(), c["rows"], row_stride=(nh + 2 * nk) * D,
                   stream=stream)
    if kind in ("kv", "load"):
        K.kv_load(s["cache"], typ, s["k_out"].data_ptr(), s["v_out"].data_ptr(), c["rows"], slots=s["slots"].data_ptr(),
                  stream=stream)
        return s["k_out"], s["v_out"]
    if kind == "tree":
        K.attention_tree(s["cache"], typ, s["q"].data_ptr(), s["out"].data_ptr(), c["n_head"], c["drafts"],
                         s["prefix"].data_ptr(), s["max_prefix"], s["workspace"], counts=s["count"].data_ptr(),
                         mask=s["mask"].data_ptr(), stream=stream)
        return s["out"]
    K.token_logprobs(typ, s["x"].data_ptr(), c["rows"], c["vocab"], s["workspace"], tokens=s["tokens"].data_ptr(),
                     logprob=s["logprob"].data_ptr(), entropy=s["entropy"].data_ptr(), n_top=c["top"],
                     top_idx=s["top_idx"].data_ptr(), top_logprob=s["top_logprob"].data_ptr(),
                     temperature=c["temperature"], row_stride=c["stride"], stream=stream)
    return {n: s[n] for n in ("logprob", "entropy", "top_idx", "top_logprob")}


# ------------------------------------------------------------------ one pass in plain torch

def _rope_plain(x, w, cos, sin, c):
    """Heads x [rows][heads][D] in float32, normalised and rotated."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    n = c["n_rot"]
    rot, rest = x[..., :n], x[..., n:]
    cos, sin = cos[:, None], sin[:, None]
    if c["layout"] == "half":
        a, b = rot[..., :n // 2], rot[..., n // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1)
    a, b = rot[..., 0::2], rot[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), rest], -1)


def _seen(s, c, L):
    """[n_seq][drafts][L]: the slots each draft attends to."""
    T = c["drafts"]
    slot = torch.arange(L, device="cuda")
    u = slot[None] - s["prefix"][:, None].long()  # [n_seq][L]: the draft in a slot
    bit = torch.arange(T, device="cuda")
    bits = (s["mask"][:, :, bit // 64] >> (bit % 64)) & 1  # [n_seq][T][T]
    inside = (u >= 0) & (u < s["count"][:, None])
    drafts = torch.gather(bits, 2, u.clamp(0, T - 1)[:, None, :].expand(-1, T, -1)).bool()
    return (u < 0)[:, None] | (drafts & inside[:, None])


def _run_plain(s, c):
    kind, dt = c["kind"], TYPES[c["type"]]
    if kind == "rope":
        nh, nk, D = c["n_head"], c["n_head_kv"], c["head_dim"]
        th = s["pos"].double()[:, None] * s["inv"][None]
        cos, sin = (torch.cos(th) * s["mscale"]).float(), (torch.sin(th) * s["mscale"]).float()
        x = s["qkv"].view(c["rows"], nh + 2 * nk, D)
        q = _rope_plain(x[:, :nh].float(), s["q_norm"], cos, sin, c)
        k = _rope_plain(x[:, nh:nh + nk].float(), s["k_norm"], cos, sin, c)
        return q.to(dt).flatten(1), k.to(dt).flatten(1)
    if kind in ("kv", "load"):
        n, nh, nk, D, T = c["n_seq"], c["n_head"], c["n_head_kv"], c["head_dim"], c["rows"]
        seq, slot = torch.arange(n, device="cuda")[:, None], s["slots"].long()
        if kind == "kv":
            x = s["qkv"].view(n, T, nh + 2 * nk, D)
            for name, part in (("k", x[:, :, nh:nh + nk]), ("v", x[:, :, nh + nk:])):
                code, scale = _quantise(part.float(), c["format"])
                s[name].view(torch.int8 if c["format"] != "f16" else torch.float16)[seq, :, slot] = \
                    code.view(torch.int8 if c["format"] != "f16" else torch.float16)
                if scale is not None:
                    s[name + "_scale"][seq, :, slot] = scale
        out = []
        for name in ("k", "v"):
            raw = s[name].view(torch.int8) if c["format"] == "f8" else s[name]
            code, scale = raw[seq, :, slot], s[name + "_scale"]
            if c["format"] == "f8":
                code = code.view(torch.float8_e4m3fn)
            out.append(_values(code, None if scale is None else scale[seq, :, slot]).to(dt).reshape(n * T, nk * D))
        return tuple(out)
    if kind == "tree":
        n, nh, nk, D, T = c["n_seq"], c["n_head"], c["n_head_kv"], c["head_dim"], c["drafts"]
        G, L = nh // nk, s["max_prefix"] + T
        kv = [_values(s[m][:, :, :L], None if s[m + "_scale"] is None else s[m + "_scale"][:, :, :L]) for m in ("k", "v")]
        q = s["q"].view(n, T, nk, G, D).permute(0, 2, 1, 3, 4).reshape(n, nk, T * G, D).float()
        scores = torch.matmul(q, kv[0].transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
        seen = _seen(s, c, L)[:, None, :, None].expand(n, nk, T, G, L).reshape(n, nk, T * G, L)
        scores = scores.masked_fill(~seen, -math.inf)
        e = torch.exp(scores - scores.amax(-1, keepdim=True))
        o = torch.matmul(e / e.sum(-1, keepdim=True), kv[1])
        o = o.view(n, nk, T, G, D).permute(0, 2, 1, 3, 4).reshape(n, T, nh * D)
        live = torch.arange(T, device="cuda")[None] < s["count"][:, None]
        return torch.where(live[..., None], o, torch.zeros_like(o)).to(dt).view(n * T, nh * D)
    raw = s["x"][:, :c["vocab"]].float()
    x = raw / c["temperature"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    l = e.sum(-1, keepdim=True)
    lse = m + torch.log(l)
    d = torch.where(e > 0, d, torch.zeros_like(d))
    entropy = (torch.log(l) - (e * d).sum(-1, keepdim=True) / l)[:, 0]
    logprob = (torch.gather(x, 1, s["tokens"].long()[:, None]) - lse)[:, 0]
    # the largest logits, ties to the lowest index: ordered bits of the value above the reversed index
    b = (raw + 0.0).view(torch.int32)
    key = ((b ^ ((b >> 31) & 0x7FFFFFFF)).long() << 32) | (0xFFFFFFFF - torch.arange(c["vocab"], device="cuda"))
    idx = 0xFFFFFFFF - (torch.topk(key, c["top"], dim=-1).values & 0xFFFFFFFF)
    return dict(logprob=logprob, entropy=entropy, top_idx=idx.to(torch.int32), top_logprob=torch.gather(x, 1, idx) - lse)


def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c, kind = case, case["kind"]
    size = 4 if c["type"] == "f32" else 2
    if kind == "rope":
        n = c["rows"] * (c["n_head"] + c["n_head_kv"]) * c["head_dim"]
        return dict(bytes=2 * size * n + 4 * c["rows"], flops=(3.0 + 4.0 * c["norm"]) * n)
    if kind == "logprobs":
        return dict(bytes=c["rows"] * (size * c["vocab"] + 12 + 8 * c["top"]), flops=5.0 * c["rows"] * c["vocab"])
    nk, D = c["n_head_kv"], c["head_dim"]
    slot = 2 * nk * (2 * D if c["format"] == "f16" else D + 4)  # a slot's keys and values, all heads
    if kind in ("kv", "load"):
        rows = c["n_seq"] * c["rows"]
        io = 2 * nk * D * size
        return dict(bytes=rows * ((2 if kind == "kv" else 1) * (slot + io) + 4),
                    flops=(4.0 if kind == "kv" else 1.0) * rows * 2 * nk * D)
    # (of a ragged batch: the sequences' mean prefix and drafts)
    prefix = c["prefix"] * (0.875 if c["ragged"] else 1.0)
    drafts = c["drafts"] * (0.5 if c["ragged"] else 1.0)
    rows = c["n_seq"] * drafts
    return dict(bytes=c["n_seq"] * (prefix + drafts) * slot + rows * (2 * c["n_head"] * D * size + 8),
                flops=4.0 * rows * c["n_head"] * D * (prefix + drafts / 2))


# ------------------------------------------------------------------ the definitions in 64 bits

def _kv64(x, form):
    """Rows in float64 as a cache of the format holds them."""
    if form == "f16":
        return x.to(torch.float16).double()
    top = 127.0 if form == "i8" else 448.0
    amax = x.abs().amax(-1, keepdim=True)
    unit = (amax / top).clamp_min(1e-300)
    y = x * top / amax.clamp_min(1e-300)
    if form == "i8":
        return torch.round(y) * unit
    # e4m3: three bits after the leading one, steps of 2^-9 below 2^-6
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step * unit


def _tree64(c, seed):
    """The attention case in float64, draft by draft."""
    c = dict(c, n_ctx=c["prefix"] + c["drafts"] + 33)
    prefix, count, sees = _tree(c, seed)
    s = _filled_cache(c, seed)
    n, nh, nk, D, T = c["n_seq"], c["n_head"], c["n_head_kv"], c["head_dim"], c["drafts"]
    G = nh // nk
    q = (1.5 * _randn(_gen(seed, 4), (n * T, nh * D))).to(TYPES[c["type"]]).double().view(n, T, nk, G, D)
    out = torch.zeros((n, T, nk, G, D), dtype=torch.float64, device="cuda")
    for i in range(n):
        P, N = int(prefix[i]), int(count[i])
        if N == 0:
            continue
        tree = torch.from_numpy(sees[i, :N, :N]).cuda()
        for h in range(nk):
            kk, vv = (s[m][i, h, :P + N].float().double() if s[m + "_scale"] is None else
                      s[m][i, h, :P + N].float().double() * s[m + "_scale"][i, h, :P + N].double()[:, None]
                      for m in ("k", "v"))
            for g in range(G):
                a = q[i, :N, h, g] @ kk.T.contiguous() / math.sqrt(D)
                a[:, P:].masked_fill_(~tree, -math.inf)
                out[i, :N, h, g] = torch.softmax(a, -1) @ vv
    return out.view(n * T, nh * D)


def exact(case, seed):
    c, kind = case, case["kind"]
    if kind == "rope":
        s = _rope_inputs(c, seed)
        nh, nk, D, n = c["n_head"], c["n_head_kv"], c["head_dim"], c["n_rot"]
        z = torch.exp(1j * (s["pos"].double()[:, None] * s["inv"])) * s["mscale"]
        out = []
        for first, heads, w in ((0, nh, s["q_norm"]), (nh, nk, s["k_norm"])):
            x = s["qkv"].view(-1, nh + 2 * nk, D)[:, first:first + heads].double()
            if w is not None:
                x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS) * w.double()
            y = x.clone()
            i, j = (slice(0, n // 2), slice(n // 2, n)) if c["layout"] == "half" else (slice(0, n, 2), slice(1, n, 2))
            t = torch.complex(x[..., i], x[..., j]) * z[:, None]
            y[..., i], y[..., j] = t.real, t.imag
            out.append(y.flatten(1))
        return tuple(out)
    if kind == "kv":
        s = _kv_inputs(c, seed)
        nh, nk, D = c["n_head"], c["n_head_kv"], c["head_dim"]
        x = s["qkv"].view(-1, nh + 2 * nk, D).double()
        return tuple(_kv64(x[:, a:a + nk], c["format"]).flatten(1) for a in (nh, nh + nk))
    if kind == "load":
        s = _filled_cache(c, seed)
        slots = _load_slots(c, seed)
        out = []
        for name in ("k", "v"):
            rows = []
            for i in range(c["n_seq"]):
                at = torch.from_numpy(slots[i]).long().cuda()
                x = (s[name][i].to(torch.float16) if c["format"] == "f8" else s[name][i])[:, at].double()
                if s[name + "_scale"] is not None:
                    x = x * s[name + "_scale"][i][:, at].double()[..., None]
                rows.append(x.permute(1, 0, 2).flatten(1))
            out.append(torch.cat(rows))
        return tuple(out)
    if kind == "tree":
        return _tree64(c, seed)
    s = _logit_inputs(c, seed)
    out = dict(logprob=[], entropy=[], top_idx=[], top_logprob=[])
    for i in range(0, c["rows"], 32):
        raw = s["x"][i:i + 32, :c["vocab"]].double()
        x = raw / c["temperature"]
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        p = torch.exp(lp)
        out["entropy"].append(-torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1))
        out["logprob"].append(torch.gather(lp, 1, s["tokens"][i:i + 32].long()[:, None])[:, 0])
        order = torch.sort(raw, dim=-1, descending=True, stable=True).indices[:, :c["top"]]
        out["top_idx"].append(order.to(torch.int32))
        out["top_logprob"].append(torch.gather(lp, 1, order))
    return {n: torch.cat(v) for n, v in out.items()}
