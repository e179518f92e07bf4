"""Serving many requests from a paged cache held in 4 bits, as cases that can be timed and checked.

Three operators, one attention layer of a model each time:

``tables``  a scheduling step: from the requests' lengths and the tokens that each
            adds (or, where it ends, gives back), the pages of its block table, the
            slots and positions of the new tokens, and the stack of free pages.
``append``  the new tokens' keys and values are quantised into their slots, and
            read back as the cache holds them (what ``update_and_fetch`` returns).
``attend``  the new tokens' queries over all tokens of their requests: decode
            steps, speculative verification, prompts, chunks of long prompts, and
            batches that mix these.

Sizes are those of the package's benchmark and tests (32 query / 8 KV heads of 128
dims, 16 / 4 of 64; 509 to 131072 tokens; batches of 1 to 16) and odd ones around
them; pages of 16 to 128 tokens, groups of 32 to 128 dims.

A page holds, for each KV head (P tokens, D dims, G = D / group groups):
  k_codes int32 [P][D/8]    dim 8w+j of a token at bit 4*(j//2) + 16*(j%2) of word w
  v_codes int32 [P/8][D]    token 8w+j at that bit of word [w][d]
  k_meta, v_meta [G][P][2]  scale and zero of a token's group, in the cache's type
"""

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 1 << 25      # elements quantised at a time
PAD = 5              # rows behind the last request in a padded batch


def _package():
    import __graft_entry__
    return __graft_entry__.load_package()


def _case(name, kind, shape, b, t, new, hq=32, hkv=8, d=128, group=64, page=64, dtype="fp16",
          pad=False):
    c = dict(kind=kind, shape=shape, b=b, t=t, new=new, hq=hq, hkv=hkv, d=d, group=group,
             page=page, dtype=dtype, pad=pad)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one interactive request takes its next token: latency alone
        _case("tables_b1_t509", "tables", "step", 1, 509, 1),
        # a server's decode step: 256 requests, some of them ending
        _case("tables_b256_t32768", "tables", "step", 256, 32768, 1, page=16),
        # 61 requests enter with their whole prompts
        _case("tables_prompts_b61_t8003", "tables", "prompt", 61, 0, 8003, pad=True),
        # the tokens of a decode step of 16 requests
        _case("append_step_b16", "append", "step", 16, 4099, 1, dtype="bf16"),
        # the encoder's bulk size: 8 heads x 8192 tokens
        _case("append_prompt_t8192", "append", "prompt", 1, 0, 8192, page=128),
        # prompts of odd lengths of a model with 64-dim heads
        _case("append_prompts_d64_b7_t2041", "append", "prompt", 7, 0, 2041, hq=16, hkv=4, d=64,
              group=32, page=16, dtype="bf16", pad=True),
        # an interactive chat early in its context
        _case("attend_step_t509", "attend", "step", 1, 509, 1),
        # one long-context stream
        _case("attend_step_t32768", "attend", "step", 1, 32768, 1),
        # a server batch of uneven requests, bfloat16
        _case("attend_step_b8_t32768", "attend", "step", 8, 32768, 1, page=16, dtype="bf16"),
        # four drafted tokens verified, 64-dim heads in groups of 32
        _case("attend_spec_d64_b2_t6001", "attend", "step", 2, 6001, 4, hq=16, hkv=4, d=64,
              group=32, page=32),
        # a whole prompt, odd length
        _case("attend_prompt_t4093", "attend", "prompt", 1, 0, 4093),
        # two chunks of long prompts beside six decode steps
        _case("attend_mixed_b8_t8192_n512", "attend", "mixed", 8, 8192, 512, dtype="bf16",
              pad=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    hq, hkv = rng.choice([(32, 8), (32, 8), (32, 8), (8, 2), (16, 2), (16, 16), (28, 4), (16, 4)])
    d, group = rng.choice([(128, 64), (128, 64), (128, 128), (128, 32), (64, 64), (64, 32)])
    kw = dict(hq=hq, hkv=hkv, d=d, group=group, page=rng.choice([16, 32, 64, 128]),
              dtype=rng.choice(["fp16", "bf16"]), pad=rng.random() < 0.3)
    kind = rng.choice(["tables", "append", "append", "attend", "attend", "attend", "attend"])
    if kind == "tables":
        b = _log_int(rng, 1, 256)
        if rng.random() < 0.5:
            return _case(None, kind, "step", b, _log_int(rng, 16, 32768), rng.choice([1, 1, 4]), **kw)
        return _case(None, kind, "prompt", b, 0, _log_int(rng, 16, 131072 // b), **kw)
    if kind == "append":
        if rng.random() < 0.4:
            b = _log_int(rng, 1, 256)
            return _case(None, kind, "step", b, _log_int(rng, 16, min(8192, 262144 // b)),
                         rng.choice([1, 1, 4]), **kw)
        b = rng.choice([1, 2, 7])
        return _case(None, kind, "prompt", b, 0, _log_int(rng, 16, 8192 * 8 // (b * hkv)), **kw)
    shape = rng.choice(["step", "step", "step", "prompt", "mixed"])
    b = rng.choice([1, 1, 2, 4, 8, 16])
    if shape == "step":
        return _case(None, kind, shape, b, _log_int(rng, 16, min(131072, 262144 * 8 // (b * hkv))),
                     rng.choice([1, 1, 1, 2, 4, 7]), **kw)
    if shape == "prompt":
        b = rng.choice([1, 1, 2, 3])
        return _case(None, kind, shape, b, 0, _log_int(rng, 16, 4093 // b), **kw)
    b = rng.choice([2, 4, 8])
    return _case(None, kind, shape, b, _log_int(rng, 200, 65536 // b), _log_int(rng, 16, 512), **kw)


# ------------------------------------------------------------------- inputs


def _requests(c):
    """(tokens held, tokens added) of every request: the first the longest,
    the others shorter by up to eight times (a prompt by four).  In a step of
    more than 8 requests one in 16 ends: it adds minus what it holds."""
    r = random.Random(c["b"] * 1000003 + c["t"] * 31 + c["new"])
    b, t, n = c["b"], c["t"], c["new"]
    if c["shape"] == "prompt":
        return [0] * b, [n] + [max(1, int(n * r.uniform(0.25, 1))) for _ in range(b - 1)]
    held = [t] + [max(1, int(t * r.uniform(0.125, 1))) for _ in range(b - 1)]
    if c["shape"] == "mixed":
        return held, [n if i < max(1, b // 4) else 1 for i in range(b)]
    if c["kind"] == "tables" and b > 8:
        return held, [-h if i % 16 == 9 else n for i, h in enumerate(held)]
    return held, [n] * b


def _rows(c):
    return sum(max(0, n) for n in _requests(c)[1]) + (PAD if c["pad"] else 0)


def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt) % (1 << 62))


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pages(c, held, seed, spare):
    """Block table of the requests over a pool in random order, and the
    stack of the pages left over (its entries behind n_free are stale)."""
    page = c["page"]
    have = [-(-h // page) for h in held]
    end = [-(-(h + max(0, n)) // page) for h, n in zip(held, _requests(c)[1])]
    total = sum(max(a, b) for a, b in zip(have, end)) + spare
    order = torch.randperm(total, generator=_gen(seed, 1), device="cuda").to(torch.int32)
    width = max(max(end), max(have), 1)
    first = torch.tensor([0] + have, device="cuda").cumsum(0)[:-1]
    col = torch.arange(width, device="cuda")
    used = col[None, :] < torch.tensor(have, device="cuda")[:, None]
    at = (first[:, None] + col[None, :]).clamp(max=total - 1)
    table = torch.where(used, order[at], torch.full_like(order[at], -1))
    left = total - sum(have)
    free = torch.zeros(total, dtype=torch.int32, device="cuda")
    free[:left] = order[sum(have):]
    return table, free, _ints([left]), total


def _filled(c, n_pages, seed):
    """A pool of pages that hold tokens: anisotropic keys, unit values."""
    dt, d, g = DTYPES[c["dtype"]], c["d"], c["d"] // c["group"]
    hkv, page = c["hkv"], c["page"]
    gen = _gen(seed, 3)
    s = 0.5 + 3.5 * torch.rand((d,), generator=gen, device="cuda")
    kc = torch.empty((n_pages, hkv, page, d // 8), dtype=torch.int32, device="cuda")
    vc = torch.empty((n_pages, hkv, page // 8, d), dtype=torch.int32, device="cuda")
    km = torch.empty((n_pages, hkv, g, page, 2), dtype=dt, device="cuda")
    vm = torch.empty_like(km)
    per = max(1, CHUNK // (hkv * page * d))
    for i in range(0, n_pages, per):
        n = min(per, n_pages - i)
        k = (torch.randn((n, hkv, page, d), generator=gen, device="cuda") * s).to(dt)
        v = torch.randn((n, hkv, page, d), generator=gen, device="cuda").to(dt)
        kq, km[i:i + n] = _quantized(k, c["group"], (0, 1, 3, 2, 4))
        vq, vm[i:i + n] = _quantized(v, c["group"], (0, 1, 3, 2, 4))
        kc[i:i + n] = _packed(kq.unflatten(-1, (-1, 8)))
        vc[i:i + n] = _packed(vq.unflatten(2, (-1, 8)).transpose(3, 4))
    return s, [kc, vc, km, vm]


def prepare(case, seed):
    c = case
    held, new = _requests(c)
    dt, n = DTYPES[c["dtype"]], _rows(c)
    st = {"case": c, "new": _ints(new), "rows": n}
    if c["kind"] == "tables":
        table, free, n_free, _ = _pages(c, held, seed, 8)
        return dict(st, lengths=_ints(held), table=table, free=free, n_free=n_free)
    after = [h + x for h, x in zip(held, new)]
    table, _, _, total = _pages(dict(c, kind="append"), after, seed, 3)
    starts = torch.tensor([0] + new, device="cuda").cumsum(0)
    st["starts"] = starts.to(torch.int32)
    s, st["store"] = _filled(c, total, seed)
    gen = _gen(seed, 4)
    if c["kind"] == "append":
        # the slots of the new tokens, as the scheduling step gives them
        tok = torch.arange(n, device="cuda")
        req = (torch.searchsorted(starts, tok, right=True) - 1).clamp(max=len(new) - 1)
        pos = torch.tensor(held, device="cuda")[req] + tok - starts[req]
        real = tok < starts[-1]
        col = torch.where(real, pos // c["page"], 0)
        slot = table[req, col].long() * c["page"] + pos % c["page"]
        st["slots"] = torch.where(real, slot, -1).to(torch.int32)
        shape = (n, c["hkv"], c["d"])
        st["k"] = (torch.randn(shape, generator=gen, device="cuda") * s).to(dt)
        st["v"] = torch.randn(shape, generator=gen, device="cuda").to(dt)
        return st
    st["q"] = torch.randn((n, c["hq"], c["d"]), generator=gen, device="cuda").to(dt)
    return dict(st, table=table, lengths=_ints(after), scale=1.0 / math.sqrt(c["d"]),
                max_new=max(new), max_length=max(after))


# -------------------------------------------------------------- plain forms


def _shifts():
    j = torch.arange(8, dtype=torch.int32, device="cuda")
    return 4 * (j // 2) + 16 * (j % 2)


def _packed(codes):
    """(..., 8) codes -> their int32 words."""
    return (codes.to(torch.int32) << _shifts()).sum(-1, dtype=torch.int32)


def _unpacked(words):
    """int32 words -> (..., 8) codes as float32."""
    return ((words[..., None] >> _shifts()) & 15).float()


def _quantized(x, group, order):
    """Codes of (..., D) rows, and each group's scale and zero, (..., G, 2)
    with its axes in `order`."""
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((hi - lo) / 15.0).to(x.dtype).float()
    code = torch.round((g - lo) / torch.where(scale > 0, scale, 1.0)).clamp(0, 15)
    code = torch.where(scale > 0, code, 0.0).flatten(-2)
    meta = torch.cat((scale, lo), -1).to(x.dtype)
    return code, meta.permute(order)


def _tables(s):
    page = s["case"]["page"]
    table, free = s["table"], s["free"]
    length, n = s["lengths"].long(), s["new"].long()
    after = length + n
    held, want = (length + page - 1) // page, (after + page - 1) // page
    give, take = (held - want).clamp(min=0), (want - held).clamp(min=0)
    given, taken = give.cumsum(0), take.cumsum(0)
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    # freed pages onto the stack, in the order of requests and pages
    back = (col >= want[:, None]) & (col < held[:, None])
    at = s["n_free"].long() + (given - give)[:, None] + col - want[:, None]
    stack = torch.cat((free, free[:1]))
    stack.index_copy_(0, torch.where(back, at, free.numel()).flatten(), table.flatten())
    free.copy_(stack[:-1])
    # new pages from its top
    top = s["n_free"].long() + given[-1]
    more = (col >= held[:, None]) & (col < want[:, None])
    at = top - 1 - ((taken - take)[:, None] + col - held[:, None])
    table.copy_(torch.where(more, free[at.clamp(0, free.numel() - 1)], table))
    # the new tokens, packed request after request
    starts = torch.cat((n.new_zeros(1), n.clamp(min=0).cumsum(0)))
    tok = torch.arange(s["rows"], device="cuda")
    req = (torch.searchsorted(starts, tok, right=True) - 1).clamp(max=n.numel() - 1)
    pos = length[req] + tok - starts[req]
    real = tok < starts[-1]
    slot = table[req, torch.where(real, pos // page, 0)].long() * page + pos % page
    i32 = torch.int32
    return {"table": table, "free": free, "n_free": (top - taken[-1]).to(i32).reshape(1),
            "lengths": after.to(i32), "starts": starts.to(i32),
            "slots": torch.where(real, slot, -1).to(i32),
            "positions": torch.where(real, pos, -1).to(i32)}


def _write(place, words, real):
    """Adds to int32 words the difference to what they shall hold (each of
    the bits is written once; rows behind the requests write nothing)."""
    flat, at = place
    delta = torch.where(real, words - flat[at], 0)
    flat.index_put_((at,), delta, accumulate=True)


def _append(s):
    c = s["case"]
    kc, vc, km, vm = s["store"]
    page, hkv, d, group = c["page"], c["hkv"], c["d"], c["group"]
    slot = s["slots"].long()
    real = (slot >= 0)[:, None, None]
    slot = slot.clamp(min=0)
    row = (slot // page)[:, None] * hkv + torch.arange(hkv, device="cuda")  # (N, H)
    off = (slot % page)[:, None, None]
    word, dim = torch.arange(d // 8, device="cuda"), torch.arange(d, device="cuda")
    grp = torch.arange(d // group, device="cuda")
    kq, kmeta = _quantized(s["k"], group, (0, 1, 2, 3))
    vq, vmeta = _quantized(s["v"], group, (0, 1, 2, 3))
    at_k = (row[..., None] * page + off) * (d // 8) + word
    _write((kc.view(-1), at_k), _packed(kq.unflatten(-1, (-1, 8))), real)
    at_v = (row[..., None] * (page // 8) + off // 8) * d + dim
    shift = _shifts()[off % 8]
    old = (vc.view(-1)[at_v] >> shift) & 15
    delta = torch.where(real, (vq.to(torch.int32) - old) << shift, 0)
    vc.view(-1).index_put_((at_v,), delta, accumulate=True)
    at_m = (row[..., None] * (d // group) + grp) * page + off
    for meta, place in ((kmeta, km), (vmeta, vm)):
        pair = meta.contiguous().view(torch.int32)[..., 0]
        _write((place.view(torch.int32).view(-1), at_m), pair, real)
    # read back
    k = _unpacked(kc.view(-1)[at_k]).flatten(-2).unflatten(-1, (-1, group))
    v = ((vc.view(-1)[at_v] >> shift) & 15).float().unflatten(-1, (-1, group))
    out = {}
    for name, code, place in (("k", k, km), ("v", v, vm)):
        m = place.view(-1, 2)[at_m].float()
        x = (m[..., 1:] + code * m[..., :1]).flatten(-2)
        out[name] = torch.where(real, x, 0.0).to(s["k"].dtype)
    return out


def _held(s):
    """Every request's keys and values, (R, H, T, D) float32."""
    c = s["case"]
    kc, vc, km, vm = s["store"]
    cols = -(-s["max_length"] // c["page"])
    pages = s["table"][:, :cols].long().clamp(min=0)
    k = _unpacked(kc[pages]).flatten(-2)                       # (R, C, H, P, D)
    v = _unpacked(vc[pages]).transpose(-1, -2).flatten(3, 4)
    both = []
    for code, meta in ((k, km), (v, vm)):
        m = meta[pages].float().transpose(3, 4)                # (R, C, H, P, G, 2)
        x = m[..., 1:] + code.unflatten(-1, (-1, c["group"])) * m[..., :1]
        both.append(x.flatten(-2).transpose(1, 2).flatten(2, 3))
    return both


def _attend(s):
    c = s["case"]
    rep = c["hq"] // c["hkv"]
    k, v = _held(s)
    starts, length = s["starts"].long(), s["lengths"].long()
    n = starts[1:] - starts[:-1]
    i = torch.arange(s["max_new"], device="cuda")
    rows = (starts[:-1, None] + i).clamp(max=s["rows"] - 1)
    q = s["q"].float()[rows]                                   # (R, M, Hq, D)
    q = q.unflatten(2, (c["hkv"], rep)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * s["scale"]
    pos = (length - n)[:, None] + i
    key = torch.arange(k.shape[2], device="cuda")
    seen = (key <= pos[..., None]) & (key < length[:, None, None])  # (R, M, T)
    score = score.unflatten(2, (rep, -1)).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, 0.0)).flatten(2, 3)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    out = out.unflatten(2, (rep, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # (R, M, Hq, D)
    tok = torch.arange(s["rows"], device="cuda")
    req = (torch.searchsorted(starts, tok, right=True) - 1).clamp(max=n.numel() - 1)
    real = (tok < starts[-1])[:, None, None]
    out = out[req, (tok - starts[req]).clamp(max=s["max_new"] - 1)]
    return torch.where(real, out, 0.0).to(s["q"].dtype)


# ---------------------------------------------------------------- the calls


def run(state):
    s = state
    kind = s["case"]["kind"]
    if not own:
        return {"tables": _tables, "append": _append, "attend": _attend}[kind](s)
    S = _package()
    if kind == "tables":
        plan = S.build_block_tables(s["lengths"], s["new"], s["table"], s["free"], s["n_free"],
                                    s["case"]["page"], s["rows"])
        return {"table": s["table"], "free": s["free"], "n_free": plan.n_free,
                "lengths": plan.lengths, "starts": plan.token_starts, "slots": plan.slots,
                "positions": plan.positions}
    store = S.PagedKVStore(*s["store"])
    if kind == "append":
        S.append_paged(store, s["k"], s["v"], s["slots"])
        k, v = S.read_paged(store, s["slots"])
        return {"k": k, "v": v}
    return S.paged_attention(s["q"], store, s["table"], s["lengths"], s["starts"], s["scale"],
                             max_new=s["max_new"], max_length=s["max_length"])


# ------------------------------------------------------------ what it takes


def work(case):
    c = case
    held, new = _requests(c)
    rows = sum(max(0, n) for n in new)
    token = c["hkv"] * (c["d"] + 8 * (c["d"] // c["group"]))  # stored bytes of a token
    if c["kind"] == "tables":
        moved = sum(abs(-(-(h + n) // c["page"]) - -(-h // c["page"])) for h, n in zip(held, new))
        return {"bytes": 16 * len(new) + 8 * moved + 8 * _rows(c), "flops": 0}
    if c["kind"] == "append":
        raw = 4 * c["hkv"] * c["d"]
        return {"bytes": rows * (2 * raw + 2 * token + 4), "flops": 20 * rows * c["hkv"] * c["d"]}
    pairs = sum(n * h + n * (n + 1) // 2 for h, n in zip(held, new))
    read = sum(h + n for h, n in zip(held, new)) * token
    return {"bytes": read + 4 * rows * c["hq"] * c["d"], "flops": 4 * pairs * c["hq"] * c["d"]}


# --------------------------------------------------------------- in 64 bits


def _bits(words):
    """Codes of int32 words as a list over their eight places."""
    return [((words >> (4 * (j >> 1) + 16 * (j & 1))) & 15).double() for j in range(8)]


def _quantized64(x, group):
    """What the cache holds of (..., D) rows, in 64 bits."""
    x64 = x.double().reshape(*x.shape[:-1], -1, group)
    zero = x64.min(-1, keepdim=True).values
    step = ((x64.max(-1, keepdim=True).values - zero) / 15).to(x.dtype).double()
    code = ((x64 - zero) / step.clamp(min=1e-300)).round().clamp(0, 15)
    return (zero + code * step).reshape(x.shape)


def exact(case, seed):
    c = case
    if c["kind"] == "tables":
        return None
    s = prepare(c, seed)
    if c["kind"] == "append":
        real = (s["slots"] >= 0).double()[:, None, None]
        return {x: _quantized64(s[x], c["group"]) * real for x in ("k", "v")}
    kc, vc, km, vm = s["store"]
    held, new = _requests(c)
    rep = c["hq"] // c["hkv"]
    out = torch.zeros((s["rows"], c["hq"], c["d"]), dtype=torch.float64, device="cuda")
    first = 0
    for r, (h, n) in enumerate(zip(held, new)):
        total = h + n
        ids = s["table"][r, :-(-total // c["page"])].long()
        for kv in range(c["hkv"]):
            k = torch.stack(_bits(kc[ids, kv]), -1).reshape(-1, c["d"])[:total]
            v = torch.stack(_bits(vc[ids, kv]), 2).reshape(-1, c["d"])[:total]
            x = []
            for code, meta in ((k, km), (v, vm)):
                m = meta[ids, kv].double()                      # (C, G, P, 2)
                step = m[..., 0].permute(0, 2, 1).reshape(-1, c["d"] // c["group"])[:total]
                zero = m[..., 1].permute(0, 2, 1).reshape(-1, c["d"] // c["group"])[:total]
                x.append(code * step.repeat_interleave(c["group"], 1)
                         + zero.repeat_interleave(c["group"], 1))
            late = torch.arange(total, device="cuda")[None, :] > \
                h + torch.arange(n, device="cuda")[:, None]
            for hq in range(kv * rep, (kv + 1) * rep):
                score = (s["q"][first:first + n, hq].double() @ x[0].t()) * s["scale"]
                w = torch.softmax(score.masked_fill(late, -math.inf), -1)
                out[first:first + n, hq] = w @ x[1]
        first += n
    return out
