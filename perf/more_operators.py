"""Prompts over a paged KV cache, caches of latent vectors and the pages themselves, as cases that
can be timed and compared with 64-bit results: attention of chunks of new tokens over a cache in
bf16 or 8 bits; appending to a cache that holds one latent vector a token for all heads, and attention
over it; copying pages, forking rows (beams, parallel samples) and compacting a cache.

A case is a dict of plain values:

    name    (listed cases)
    op      "prefill": attention of every row's newest tokens over its cached keys, their own included
            "latent": attention of every row's newest queries over a cache of latent vectors
            "latent_step": new tokens appended to that cache first, their rotary parts turned
            "copy": pages copied within every layer's cache
            "fork": rows that go on from other rows, with room for new tokens
            "compact": the pages in use moved to the front of the cache
    cache   "bf16" or "fp8" (e4m3, one power-of-two scale for each run of 32 tokens of a head); latent: bf16
    Hkv, D, page   kv heads, head dim, tokens of a page

    prefill:
    B, T, Hq  rows, the most new tokens of a row, query heads
    keys    keys that the longest row has before its new tokens
    new     "all": T tokens in every row; "ragged": 1 .. T; "mixed": T in the first row, one in the others
    packed  the rows' tokens one behind another, else padded to T each
    mask    "none", "causal" or "window" (causal, the last ``window`` keys)
    score   "none" or "alibi_softcap"

    latent, latent_step:
    B, T, H   rows, new tokens of a row, heads
    L, R      elements of a token's latent vector (key and value of every head) and of its rotary part (key only)
    keys, ragged  keys that the longest row has in all (its T newest included); rows of different lengths
    mask, window  as above
    layout    (latent_step) "half": rotary pairs (i, i + R / 2); "interleaved": (2 i, 2 i + 1)

    copy, fork, compact:
    layers  layers whose caches share the page table
    pages   pages of a layer's cache
    pairs   (copy) pages to copy
    B, N    (fork) rows before and after; (compact) B rows
    keys    tokens of the longest row
    room    (fork) tokens to make room for
    keep    share of the pages that something else holds (a prefix cache)

Cache layout: keys and values are (pages, Hkv, page, D), scales (pages, Hkv, page / 32); latent vectors
and rotary parts (pages, page, L + R).
"""
import math
import os
import random
import sys

import torch

own = False  # True: run() calls the framework's kernels

DEV = "cuda"
GROUP = 32        # tokens that share a scale
SOFTCAP = 50.0
FREE = 1 << 30    # a page that nobody uses
BASE = 10000.0    # of the rotary frequencies


def _pf():
    d = os.path.join(os.getcwd(), "pallas-flexattn_amd")
    if d not in sys.path:
        sys.path.insert(0, d)
    import pallas_flexattn
    return pallas_flexattn


def _prefill(B, T, Hq, Hkv, D, keys, cache="bf16", page=64, new="all", packed=False, mask="causal", window=0, score="none",
             **more):
    return dict(op="prefill", B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, keys=keys, cache=cache, page=page, new=new, packed=packed,
                mask=mask, window=window, score=score, **more)


def _latent(op, B, T, H, L, R, keys, page=64, ragged=False, mask="causal", window=0, layout="half", **more):
    return dict(op=op, B=B, T=T, H=H, L=L, R=R, keys=keys, page=page, ragged=ragged, mask=mask, window=window, layout=layout,
                **more)


def _pages(op, Hkv, D, page, cache, layers, pages, pairs=0, B=0, N=0, keys=0, room=0, keep=0.0, **more):
    return dict(op=op, Hkv=Hkv, D=D, page=page, cache=cache, layers=layers, pages=pages, pairs=pairs, B=B, N=N, keys=keys,
                room=room, keep=keep, **more)


def listed():
    return [
        # the last few words of a chat message behind a short history: latency
        _prefill(1, 19, 32, 8, 128, 500, name="prefill_short_bf16"),
        # a chunk in the middle of a long prompt, 8-bit cache
        _prefill(1, 1024, 32, 8, 128, 16384, cache="fp8", page=128, name="prefill_chunk_fp8_16k"),
        # a scheduler's batch: one chunk of a prompt among rows that decode, packed, mixed lengths
        _prefill(32, 1500, 32, 8, 128, 8192, cache="fp8", page=64, new="mixed", packed=True, name="prefill_mixed_packed_fp8"),
        # sliding-window layer with ALiBi and a soft-cap, ungrouped heads of 64, a padded ragged batch
        _prefill(8, 700, 16, 16, 64, 3000, page=32, new="ragged", mask="window", window=1500, score="alibi_softcap",
                 name="prefill_window_ragged_d64"),
        # the last chunk of a long document: bound by the matrix cores
        _prefill(1, 4096, 32, 8, 128, 28672, page=256, name="prefill_long_32k"),
        # one request alone, the heads that one of several GPUs holds: latency
        _latent("latent", 1, 1, 16, 512, 64, 4001, name="latent_one_4k"),
        # continuous batching with all heads: as many operations a byte as the card has
        _latent("latent", 24, 1, 128, 512, 64, 8192, page=128, ragged=True, name="latent_mixed_128_heads"),
        # speculative decoding: append three tokens a row, then attend
        _latent("latent_step", 16, 3, 32, 512, 64, 6000, ragged=True, name="latent_step_spec"),
        # a prefix's pages copied for every layer
        _pages("copy", 8, 128, 128, "fp8", 16, 300, pairs=128, name="copy_prefix_16_layers"),
        # one prompt continued by eight samples
        _pages("fork", 8, 128, 64, "bf16", 4, 256, B=1, N=8, keys=5000, room=1, name="fork_8_samples"),
        # beam search: 16 requests of four beams, re-parented at every step
        _pages("fork", 4, 64, 32, "fp8", 8, 6000, B=64, N=64, keys=1800, room=1, keep=0.05, name="fork_64_beams"),
        # a cache whose rows came and went for hours, in every layer
        _pages("compact", 8, 128, 128, "fp8", 8, 700, B=48, keys=2048, name="compact_8_layers"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["prefill"] * 4 + ["latent"] * 2 + ["latent_step"] + ["copy", "fork", "fork", "compact"])
        D, Hkv = rng.choice([32, 64, 128, 128]), rng.choice([1, 2, 4, 8, 16])
        page, cache = rng.choice([32, 64, 96, 128, 256]), rng.choice(["bf16", "fp8"])
        mask = rng.choice(["none", "causal", "causal", "causal", "window"])
        if op in ("latent", "latent_step"):
            T = rng.choice([1, 1, 1, 2, 4, 7, _log(rng, 1, 300)])
            c = _latent(op, _log(rng, 1, 64), T, rng.choice([1, 5, 8, 16, 16, 32, 64, 128]), rng.choice([128, 256, 512, 512]),
                        rng.choice([32, 64, 64]), _log(rng, max(T, 16), 32768), page=page, ragged=rng.random() < 0.7,
                        mask=mask, window=_log(rng, 32, 4096) if mask == "window" else 0,
                        layout=rng.choice(["half", "interleaved"]))
            fits = c["B"] * _width(c) * page * (c["L"] + c["R"]) <= 6e8
        elif op == "prefill":
            new = rng.choice(["all", "all", "ragged", "mixed"])
            c = _prefill(_log(rng, 1, 32), _log(rng, 1, 4096), Hkv * rng.choice([1, 2, 4, 4, 7, 8]), Hkv, D,
                         0 if rng.random() < 0.25 else _log(rng, 1, 32768), cache=cache, page=page, new=new,
                         packed=rng.random() < 0.4, mask=mask, window=_log(rng, 32, 4096) if mask == "window" else 0,
                         score=rng.choice(["none", "none", "none", "alibi_softcap"]))
            fits = _cache_pages(c) * page * Hkv * D <= 3e8
        else:
            layers = _log(rng, 1, 16)
            pages = _log(rng, 32, 8192)
            keep = rng.choice([0.0, 0.0, 0.1])
            if op == "copy":
                c = _pages(op, Hkv, D, page, cache, layers, pages, pairs=_log(rng, 1, pages // 2))
            else:
                B = _log(rng, 1, 128)
                N = _log(rng, 1, 128) if op == "fork" else 0
                keys = int(page * pages * rng.uniform(0.2, 0.7) / B)
                c = _pages(op, Hkv, D, page, cache, layers, pages, B=B, N=N, keys=max(keys, 1),
                           room=rng.choice([0, 1, 1, 300]) if op == "fork" else 0, keep=keep)
            fits = layers * pages * page * Hkv * D <= 6e8
        if fits and _cost(c) <= top:
            return c


# ---------------------------------------------------------------- what a case is made of ----
def _lens(case):
    """(keys before the new tokens, new tokens) of each row."""
    B, T, keys = case["B"], case["T"], case["keys"]
    if case["op"] != "prefill":
        r = random.Random(f"latent/{B}/{T}/{keys}")
        return [keys - T] + [int((keys - T) * (r.uniform(0.1, 1.0) if case["ragged"] else 1)) for _ in range(B - 1)], [T] * B
    r = random.Random(f"prefill/{B}/{T}/{keys}")
    before = [keys] + [int(keys * r.uniform(0.1, 1.0)) for _ in range(B - 1)]
    if case["new"] == "mixed":
        return before, [T] + [1] * (B - 1)
    return before, [T] + [r.randint(1, T) if case["new"] == "ragged" else T for _ in range(B - 1)]


def _width(case):
    """Pages of a row's table: its keys and some room."""
    return -(-(case["keys"] + case["T"] + GROUP) // case["page"])


def _cache_pages(case):
    return case["B"] * _width(case)


def _pairs(case, a, t):
    """Query-key pairs of a row with t new tokens behind `a` keys."""
    if case["mask"] == "none":
        return t * (a + t)
    if case["mask"] == "causal":
        return t * a + t * (t + 1) // 2
    return sum(min(case["window"], a + i + 1) for i in range(t))


def _span(case, at, have):
    """Keys that the query at position `at` of a row with `have` keys sees: [lo, hi)."""
    if case["mask"] == "none":
        return 0, have
    return (max(0, at - case["window"] + 1) if case["mask"] == "window" else 0), at + 1


def _page_bytes(case):
    """Bytes of a page in all layers, keys and values."""
    run = 2 if case["cache"] == "bf16" else 1 + 4 / (GROUP * case["D"])
    return 2 * case["layers"] * case["Hkv"] * case["page"] * case["D"] * run


def _rows(case):
    """A fork's or compaction's tokens per row, the table of page ids (-1: none) and the pages that others keep: the
    same for every seed but the page ids' order."""
    r = random.Random(f"rows/{case['B']}/{case['keys']}/{case['pages']}/{case['page']}")
    B, page, P = case["B"], case["page"], case["pages"]
    kept = int(P * case["keep"])
    lens = [case["keys"]] + [r.randint(0, case["keys"]) for _ in range(B - 1)]
    width = -(-(case["keys"] + case["room"]) // page) + 1
    table, n = [], 0
    for b in range(B):
        mine = -(-lens[b] // page)
        shared = 0
        if b and r.random() < 0.5:  # the row shares the beginning of the one before it
            shared = r.randint(0, min(lens[b] // page, lens[b - 1] // page))
        row = table[b - 1][:shared] if b else []
        take = min(mine - shared, P - kept - n)
        if take < mine - shared:
            lens[b] = (shared + take) * page
        row = row + list(range(n, n + take))
        n += take
        table.append(row + [-1] * (width - len(row)))
    return lens, table, kept, width


def _parents(case):
    r = random.Random(f"parents/{case['B']}/{case['N']}")
    if case["B"] == 1:
        return [0] * case["N"]
    out = []
    for i in range(case["N"]):  # beams stay near their own request; a few rows end
        out.append(-1 if r.random() < 0.05 else min(case["B"] - 1, i * case["B"] // case["N"] // 4 * 4 + r.randrange(4)))
    return out


def work(case):
    if case["op"] == "prefill":
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        before, new = _lens(case)
        run = 2 if case["cache"] == "bf16" else 1 + 4 / (GROUP * D)
        nbytes = flops = 0
        for a, t in zip(before, new):
            lo = _span(case, a, a + t)[0]
            nbytes += Hkv * (a + t - lo) * 2 * D * run + t * Hq * (4 * D + 4)
            flops += 4 * Hq * D * _pairs(case, a, t)
        return {"bytes": nbytes, "flops": flops}
    if case["op"] in ("latent", "latent_step"):
        B, T, H, L, R = (case[k] for k in ("B", "T", "H", "L", "R"))
        before, _ = _lens(case)
        nbytes = B * T * H * (2 * (2 * L + R) + 4)
        if case["op"] == "latent_step":  # (the new tokens' rows are not read again)
            nbytes += B * T * (2 * (L + R) + 2 * H * R)
        flops = 0
        for a in before:
            nbytes += 2 * (L + R) * (a + T - _span(case, a, a + T)[0])
            flops += 2 * H * (2 * L + R) * _pairs(case, a, T)
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "copy":
        return {"bytes": 2 * case["pairs"] * _page_bytes(case) + 8 * case["pairs"], "flops": 0}
    moved, entries = _moves(case)
    return {"bytes": 2 * moved * _page_bytes(case) + 8 * entries + case["pages"] * (case["keep"] > 0), "flops": 0}


def _moves(case):
    """Pages that a fork or a compaction has to copy (about: a compaction's depend on the ids' order), table entries."""
    lens, table, kept, width = _rows(case)
    if case["op"] == "fork":
        last = {}
        moved = 0
        for p in _parents(case):
            if p >= 0 and lens[p] % case["page"]:
                pid = table[p][lens[p] // case["page"]]
                moved += pid in last
                last[pid] = 1
        return moved, case["N"] * width
    used = len({x for row in table for x in row if x >= 0})
    return int(used * (1 - (used + kept) / case["pages"])), case["B"] * width


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 200


def _scale_of(amax):
    """The smallest power of two 2^e, -126 <= e <= 127, with 448 2^e >= amax."""
    m, e = torch.frexp(amax.double() / 448.0)
    e = torch.where(m == 0.5, e - 1, e).clamp(-126, 127)
    return torch.ldexp(torch.ones_like(amax, dtype=torch.float64), e).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] in ("latent", "latent_step"):
        return _prepare_latent(case, gen)
    Hkv, D, page = case["Hkv"], case["D"], case["page"]

    def rnd(*s):
        return torch.randn(*s, device=DEV, generator=gen)

    prefill = case["op"] == "prefill"
    P = _cache_pages(case) if prefill else case["pages"]
    # (keys of some channels are much larger than the others, as in trained models)
    wide = 1.0 + 3.0 * (torch.rand(Hkv, 1, D, device=DEV, generator=gen) < 0.05).float()
    caches = []
    for _ in range(1 if prefill else case["layers"]):
        layer, scales = [], []
        for spread in (wide, 1.0):
            x = rnd(P, Hkv, page, D) * spread
            if case["cache"] == "bf16":
                layer.append(x.to(torch.bfloat16))
            else:
                s = _scale_of(x.reshape(P, Hkv, -1, GROUP * D).abs().amax(-1))
                layer.append((x / s.repeat_interleave(GROUP, dim=2)[..., None]).to(torch.float8_e4m3fn))
                scales.append(s)
        caches.append(layer + scales)
    st = {"case": case, "caches": caches}
    ids = torch.randperm(P, device=DEV, generator=gen)

    def ints(x):
        return torch.tensor(x, device=DEV, dtype=torch.int32)

    if prefill:
        B, T, Hq = case["B"], case["T"], case["Hq"]
        before, new = _lens(case)
        st["table"] = ids.to(torch.int32).reshape(B, -1)
        st["after"] = ints([a + t for a, t in zip(before, new)])
        # projections give (tokens, H, D); the framework's layout is a view of it
        st["q"] = rnd(*((1, sum(new)) if case["packed"] else (B, T)), Hq, D).to(torch.bfloat16).transpose(1, 2)
        if case["packed"]:
            st["starts"] = ints([sum(new[:b]) for b in range(B + 1)])
        else:
            st["new"] = ints(new) if new != [T] * B else None
        if case["score"] == "alibi_softcap":
            st["slopes"] = torch.tensor([2.0 ** (-8.0 * h / Hq) for h in range(Hq)], device=DEV)
            if own:  # the descriptor that a program keeps
                pf = _pf()
                st["score"] = pf.compose_score_mods(pf.alibi_score_mod(Hq), pf.softcap_score_mod(SOFTCAP))
        return st
    if case["op"] == "copy":
        st["src"], st["dst"] = ids[:case["pairs"]].to(torch.int32), ids[-case["pairs"]:].to(torch.int32)
        return st
    lens, table, kept, _ = _rows(case)
    t = torch.tensor(table, device=DEV)
    st["table"] = torch.where(t >= 0, ids[t.clamp(min=0)], t).to(torch.int32)
    st["lens"] = ints(lens)
    st["keep"] = None
    if kept:
        st["keep"] = torch.zeros(P, device=DEV, dtype=torch.bool)
        st["keep"][ids[-kept:]] = True
    if case["op"] == "fork":
        st["parents"] = ints(_parents(case))
    return st


def _prepare_latent(case, gen):
    B, T, H, L, R, page = (case[k] for k in ("B", "T", "H", "L", "R", "page"))

    def rnd(*s):
        return torch.randn(*s, device=DEV, generator=gen)

    before, new = _lens(case)
    P = B * _width(case)
    # (a latent vector is a norm's output; the rotary part comes from a projection)
    st = {"case": case, "cache": rnd(P, page, L + R).to(torch.bfloat16), "scale": 1.0 / math.sqrt(L / 4 + R),
          "table": torch.randperm(P, device=DEV, generator=gen).to(torch.int32).reshape(B, -1)}
    st["lens"] = torch.tensor(before, device=DEV, dtype=torch.int32)
    st["after"] = torch.tensor([a + t for a, t in zip(before, new)], device=DEV, dtype=torch.int32)
    # a product per head gives (H, tokens, L), a projection (tokens, H, R): the framework's layout is a view of each
    st["q"] = (0.5 * rnd(H, B, T, L)).to(torch.bfloat16).transpose(0, 1)
    st["qr"] = rnd(B, T, H, R).to(torch.bfloat16).transpose(1, 2)
    if case["op"] == "latent_step":
        st["freq"] = BASE ** (-torch.arange(R // 2, device=DEV, dtype=torch.float64) * 2.0 / R)
        x = rnd(B, T, L + R).to(torch.bfloat16)  # one projection gives both parts
        st["new"], st["kr"] = x[..., :L], x[..., L:]
    return st


# ---------------------------------------------------------------- one pass ----
def run(st):
    if own:
        return _run_own(st)
    return {"prefill": _plain_prefill, "latent": _plain_latent, "latent_step": _plain_latent, "copy": _plain_copy, "fork": _plain_fork, "compact": _plain_compact}[st["case"]["op"]](st)


def _mask(pf, c):
    if c["mask"] == "none":
        return None
    return pf.causal_mask if c["mask"] == "causal" else pf.MaskSpec(left=c["window"] - 1, right=0)


def _run_own(st):
    pf = _pf()
    c = st["case"]
    if c["op"] in ("latent", "latent_step"):
        cache, qr, out = pf.LatentKVCache(st["cache"], c["L"]), st["qr"], {}
        if c["op"] == "latent_step":
            rot = pf.Rotary(st["freq"], c["layout"] == "interleaved")
            qr = pf.append_latent_cache(cache, st["new"], st["kr"], st["lens"], st["table"], rotary=rot, query_rope=qr)
            out = {"cache": st["cache"], "qr": qr}
        out["o"], out["lse"] = pf.flex_decode_latent(st["q"], qr, cache, st["scale"], st["after"], st["table"],
                                                     mask_mod=_mask(pf, c), return_lse=True)
        return out
    caches = [pf.Fp8KVCache(*x) if c["cache"] == "fp8" else tuple(x) for x in st["caches"]]
    if c["op"] == "prefill":
        o, lse = pf.flex_prefill(st["q"], caches[0], st["after"], st["table"], mask_mod=_mask(pf, c),
                                 score_mod=st.get("score"), enable_gqa=True, return_lse=True, query_lens=st.get("new"),
                                 query_starts=st.get("starts"))
        return {"o": o, "lse": lse}
    if c["op"] == "copy":
        pf.copy_kv_pages(caches, st["src"], st["dst"])
        return {"caches": st["caches"]}
    if c["op"] == "fork":
        table, lens, free = pf.fork_kv_rows(caches, st["table"], st["lens"], st["parents"], room=c["room"], keep=st["keep"])
        return {"caches": st["caches"], "table": table, "lens": lens, "free": free}
    table, used = pf.compact_kv_pages(caches, st["table"], st["lens"], keep=st["keep"])
    return {"caches": st["caches"], "table": table, "used": used}


def _token_rows(st):
    """Each row's (first token's place, tokens, keys): index of a row of q, the first token in it."""
    c = st["case"]
    before, new = _lens(c)
    at = 0
    for b, (a, t) in enumerate(zip(before, new)):
        yield (b, 0 if c["packed"] else b, at if c["packed"] else 0, t, a + t)
        at += t


def _plain_prefill(st):
    c = st["case"]
    Hq, Hkv, D, page = c["Hq"], c["Hkv"], c["D"], c["page"]
    g = Hq // Hkv
    q = st["q"]
    o = torch.zeros(q.shape, device=DEV)
    lse = torch.full(q.shape[:3], -math.inf, device=DEV)
    layer = st["caches"][0]
    for b, row, first, t, have in _token_rows(st):
        ids = st["table"][b, :-(-have // page)].long()
        kv = []
        for i in (0, 1):
            x = layer[i][ids].float()
            if c["cache"] == "fp8":
                x = x * layer[2 + i][ids].repeat_interleave(GROUP, dim=2)[..., None]
            kv.append(x.transpose(0, 1).reshape(Hkv, -1, D)[:, :have])
        key = torch.arange(have, device=DEV)
        step = max(1, int(2e8 / (Hq * have)))  # queries at a time: the scores of all heads fit in 1 GB
        for i in range(0, t, step):
            n = min(step, t - i)
            at = (have - t + i + torch.arange(n, device=DEV))[:, None]
            x = q[row, :, first + i:first + i + n].float().reshape(Hkv, g * n, D)
            s = (torch.matmul(x, kv[0].transpose(1, 2)) / math.sqrt(D)).reshape(Hq, n, have)
            if c["score"] == "alibi_softcap":
                s = s + st["slopes"][:, None, None] * (key - at).float()
                s = SOFTCAP * torch.tanh(s / SOFTCAP)
            if c["mask"] != "none":
                seen = key <= at
                if c["mask"] == "window":
                    seen = seen & (at - key < c["window"])
                s = torch.where(seen, s, -math.inf)
            m = s.amax(-1, keepdim=True)
            p = torch.exp(s - m)
            l = p.sum(-1, keepdim=True)
            y = torch.matmul((p / l).reshape(Hkv, g * n, have), kv[1])
            o[row, :, first + i:first + i + n] = y.reshape(Hq, n, D)
            lse[row, :, first + i:first + i + n] = (m + l.log())[..., 0]
    return {"o": o.to(torch.bfloat16), "lse": lse}


def _turn(x, cos, sin, layout):
    """Rotates x (float32) by the angles of its R / 2 pairs."""
    n = cos.shape[-1]
    if layout == "half":
        a, b = x[..., :n], x[..., n:]
        return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)


def _plain_latent(st):
    c = st["case"]
    B, T, H, L, R, page = (c[k] for k in ("B", "T", "H", "L", "R", "page"))
    qr, out = st["qr"], {}
    if c["op"] == "latent_step":
        at = st["lens"].long()[:, None] + torch.arange(T, device=DEV)
        angle = at.double()[..., None] * st["freq"]
        cos, sin = angle.cos().float(), angle.sin().float()
        spot = (torch.gather(st["table"].long(), 1, at // page), at % page)
        new = torch.cat((st["new"], _turn(st["kr"].float(), cos, sin, c["layout"]).to(torch.bfloat16)), dim=-1)
        st["cache"][spot] = new
        qr = _turn(qr.float(), cos[:, None], sin[:, None], c["layout"]).to(torch.bfloat16)
        out = {"cache": st["cache"], "qr": qr}
    o = torch.empty(B, H, T, L, device=DEV, dtype=torch.bfloat16)
    lse = torch.empty(B, H, T, device=DEV)
    before, _ = _lens(c)
    q = torch.cat((st["q"].float(), qr.float()), dim=-1)
    for b in range(B):
        have = before[b] + T
        x = st["cache"][st["table"][b, :-(-have // page)].long()].float().reshape(-1, L + R)[:have]
        s = (torch.matmul(q[b].reshape(H * T, L + R), x.T) * st["scale"]).reshape(H, T, have)
        if c["mask"] != "none":
            key = torch.arange(have, device=DEV)
            pos = have - T + torch.arange(T, device=DEV)[:, None]
            seen = key <= pos
            if c["mask"] == "window":
                seen = seen & (pos - key < c["window"])
            s = torch.where(seen, s, -math.inf)
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - m)
        l = p.sum(-1, keepdim=True)
        o[b] = torch.matmul((p / l).reshape(H * T, have), x[:, :L]).reshape(H, T, L).to(torch.bfloat16)
        lse[b] = (m + l.log())[..., 0]
    out["o"], out["lse"] = o, lse
    return out


def _bytes(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _copy(st, src, dst):
    for layer in st["caches"]:
        for x in layer:
            y = _bytes(x)
            y[dst] = y[src]


def _plain_copy(st):
    _copy(st, st["src"].long(), st["dst"].long())
    return {"caches": st["caches"]}


def _plain_fork(st):
    c = st["case"]
    P, page = c["pages"], c["page"]
    B, M = st["table"].shape
    parents = st["parents"].long()
    N = parents.shape[0]
    ok = (parents >= 0) & (parents < B)
    p = parents.clamp(0, B - 1)
    lens = torch.where(ok, st["lens"].long()[p].clamp(0, M * page), 0)
    t = st["table"].long()[p]
    there = (t >= 0) & (t < P)
    col = torch.arange(M, device=DEV)
    whole, b = lens // page, torch.arange(N, device=DEV)
    full = col < whole[:, None]
    # of each page: -1 where a row has all of it or others keep it, else the first row that ends in it
    holder = torch.full((P + 1,), FREE, device=DEV)
    last = torch.gather(t, 1, whole.clamp(max=M - 1)[:, None])[:, 0]
    ends = (lens % page > 0) & (last >= 0) & (last < P)
    holder.scatter_reduce_(0, torch.where(ends, last, P), b, "amin")
    holder[torch.where(full & there, t, P).flatten()] = -1
    if st["keep"] is not None:
        holder[:P] = torch.where(st["keep"], -1, holder[:P])
    copy = ends & (holder[torch.where(ends, last, P)] != b)
    free = holder[:P] == FREE
    have = (lens + page - 1) // page
    fresh = ((lens + c["room"]).clamp(max=M * page) + page - 1) // page - have
    need = copy.long() + fresh
    first = need.cumsum(0) - need
    # the free pages in ascending order, -1 behind them
    order = torch.full((P + N * M + 2,), -1, device=DEV)
    order[torch.where(free, free.cumsum(0) - 1, P + N * M + 1)] = torch.arange(P, device=DEV)
    order[P + N * M + 1] = -1
    table = torch.where(full, t, -1)
    own_last = torch.where(copy, order[first], last)
    table = torch.where((col == whole[:, None]) & (lens % page > 0)[:, None], own_last[:, None], table)
    nth = (first + copy)[:, None] + col - have[:, None]
    table = torch.where((col >= have[:, None]) & (col < (have + fresh)[:, None]), order[nth.clamp(min=0)], table)
    moved = copy & (own_last >= 0)
    _copy(st, last[moved], own_last[moved])
    return {"caches": st["caches"], "table": table.int(), "lens": lens.int(), "free": (free.sum() - need.sum()).int()}


def _plain_compact(st):
    c = st["case"]
    P, page = c["pages"], c["page"]
    t = st["table"].long()
    M = t.shape[1]
    lens = st["lens"].long().clamp(0, M * page)
    mine = torch.arange(M, device=DEV) < ((lens + page - 1) // page)[:, None]
    there = mine & (t >= 0) & (t < P)
    rows = torch.zeros(P + 1, device=DEV, dtype=torch.bool)
    rows[torch.where(there, t, P).flatten()] = True
    rows = rows[:P]
    held = rows if st["keep"] is None else rows | st["keep"]
    used = held.sum()
    page_id = torch.arange(P, device=DEV)
    movable = rows if st["keep"] is None else rows & ~st["keep"]
    src = (movable & (page_id >= used)).nonzero()[:, 0]
    dst = (~held & (page_id < used)).nonzero()[:, 0][:src.shape[0]]
    to = page_id.clone()
    to[src] = dst
    _copy(st, src, dst)
    table = torch.where(there, to[t.clamp(0, P - 1)], torch.where(mine, t, -1))
    return {"caches": st["caches"], "table": table.int(), "used": used.int()}


# ---------------------------------------------------------------- the definition, in 64 bits ----
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "prefill":
        return _exact_prefill(case, st)
    if case["op"] in ("latent", "latent_step"):
        return _exact_latent(case, st)
    layers = [[x.double() for x in layer] for layer in st["caches"]]

    def moved(pairs):
        for layer in layers:
            for x in layer:
                kept = [x[s].clone() for s, _ in pairs]
                for (_, d), y in zip(pairs, kept):
                    x[d] = y
        return layers

    if case["op"] == "copy":
        return {"caches": moved(list(zip(st["src"].tolist(), st["dst"].tolist())))}
    table, lens = st["table"].tolist(), st["lens"].tolist()
    keep = set() if st["keep"] is None else set(st["keep"].nonzero()[:, 0].tolist())
    P, page, width = case["pages"], case["page"], len(table[0])

    def ints(x):
        return torch.tensor(x, device=DEV, dtype=torch.int32)

    if case["op"] == "compact":
        rows = {x for row, n in zip(table, lens) for x in row[:-(-n // page)]}
        used = len(rows | keep)
        slots = [x for x in range(used) if x not in rows and x not in keep]
        to = dict(zip(sorted(x for x in rows - keep if x >= used), slots))
        out = [[to.get(x, x) if i < -(-n // page) else -1 for i, x in enumerate(row)] for row, n in zip(table, lens)]
        return {"caches": moved(list(to.items())), "table": ints(out), "used": ints(used)}
    # a fork, row by row: what rows have whole first, then who may go on in its last page
    new = []
    for p in st["parents"].tolist():
        n = lens[p] if 0 <= p < len(lens) else 0
        new.append((n, table[p][:n // page], table[p][n // page] if n % page else None))
    held = set(keep).union(*(set(whole) for _, whole, _ in new))
    taken, pairs, out = set(held), [], []
    stays = []
    for _, _, last in new:
        stays.append(last is not None and last not in taken)
        if last is not None:
            taken.add(last)
    free = iter([x for x in range(P) if x not in taken])
    left = P - len(taken)
    for (n, whole, last), mine in zip(new, stays):
        row = list(whole)
        if last is not None:
            row.append(last if mine else next(free, -1))
            if not mine:
                left -= 1
                if row[-1] >= 0:
                    pairs.append((last, row[-1]))
        while len(row) < -(-min(n + case["room"], width * page) // page):
            row.append(next(free, -1))
            left -= 1
        out.append(row + [-1] * (width - len(row)))
    return {"caches": moved(pairs), "table": ints(out), "lens": ints([n for n, _, _ in new]), "free": ints(left)}


def _exact_prefill(case, st):
    Hq, Hkv, D, page = case["Hq"], case["Hkv"], case["D"], case["page"]
    q, layer = st["q"], st["caches"][0]
    o = torch.zeros(q.shape, device=DEV, dtype=torch.float64)
    lse = torch.full(q.shape[:3], -math.inf, device=DEV, dtype=torch.float64)
    for b, row, first, t, have in _token_rows(st):
        ids = st["table"][b].long()
        k, v = (x[ids].double() for x in layer[:2])
        if case["cache"] == "fp8":
            k, v = (x * torch.repeat_interleave(s[ids].double(), GROUP, 2)[..., None] for x, s in zip((k, v), layer[2:]))
        k, v = (x.permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :have] for x in (k, v))
        for h in range(Hq):
            kh, vh = k[h * Hkv // Hq], v[h * Hkv // Hq]
            step = max(1, int(1e8 / have))
            for i in range(0, t, step):
                n = min(step, t - i)
                at = have - t + i + torch.arange(n, device=DEV)
                dist = torch.arange(have, device=DEV)[None, :] - at[:, None]
                s = q[row, h, first + i:first + i + n].double() @ kh.T * D ** -0.5
                if case["score"] == "alibi_softcap":
                    s = SOFTCAP * torch.tanh((s + st["slopes"][h].double() * dist) / SOFTCAP)
                if case["mask"] != "none":
                    s = s.masked_fill(dist > 0, -math.inf)
                if case["mask"] == "window":
                    s = s.masked_fill(dist <= -case["window"], -math.inf)
                z = torch.logsumexp(s, -1)
                lse[row, h, first + i:first + i + n] = z
                o[row, h, first + i:first + i + n] = torch.exp(s - z[:, None]) @ vh
    return {"o": o, "lse": lse}


def _exact_latent(case, st):
    B, T, H, L, R, page = (case[k] for k in ("B", "T", "H", "L", "R", "page"))
    before, _ = _lens(case)
    qr, out = st["qr"].double(), {}
    cache = st["cache"].double()
    if case["op"] == "latent_step":  # complex numbers x1 + i x2 times e^(i angle)
        j = torch.arange(R // 2, device=DEV)
        first, second = (2 * j, 2 * j + 1) if case["layout"] == "interleaved" else (j, j + R // 2)

        def turn(x, positions):
            angle = positions.double()[:, None] * st["freq"]
            w = torch.complex(x[..., first], x[..., second]) * torch.polar(torch.ones_like(angle), angle)
            y = torch.empty_like(x)
            y[..., first], y[..., second] = w.real, w.imag
            return y

        qr = qr.clone()
        for b in range(B):
            at = before[b] + torch.arange(T, device=DEV)
            k = turn(st["kr"][b].double(), at)
            qr[b] = turn(qr[b], at)
            for t in range(T):
                p = before[b] + t
                cache[int(st["table"][b, p // page]), p % page] = torch.cat((st["new"][b, t].double(), k[t]))
        out = {"cache": cache.clone(), "qr": qr}
        # what the attention reads has been rounded
        qr, cache = qr.to(torch.bfloat16).double(), cache.to(torch.bfloat16).double()
    o = torch.zeros(B, H, T, L, device=DEV, dtype=torch.float64)
    lse = torch.zeros(B, H, T, device=DEV, dtype=torch.float64)
    for b in range(B):
        have = before[b] + T
        x = cache[st["table"][b].long()].reshape(-1, L + R)[:have]
        for i in range(T):
            lo, hi = _span(case, have - T + i, have)
            s = (st["q"][b, :, i].double() @ x[lo:hi, :L].T + qr[b, :, i] @ x[lo:hi, L:].T) * st["scale"]
            z = torch.logsumexp(s, -1)
            lse[b, :, i] = z
            o[b, :, i] = torch.exp(s - z[:, None]) @ x[lo:hi, :L]
    out["o"], out["lse"] = o, lse
    return out
