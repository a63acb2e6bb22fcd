"""The operators of attention over a serving cache: their cases, their plain forms and their definitions.

All of them work on a key / value cache [batch, heads_kv, t_max, dhead] in float32, float16 or
bfloat16, with float32 queries and outputs:

  tree        ct2x_attention_tree: a tree of drafted tokens against the committed cache and itself
  accumulate  ct2x_attention_accumulate: one token per entry, its probabilities added to the weights
  evict       ct2x_cache_evict: the heaviest and the newest positions move to a smaller cache
  bounds      ct2x_cache_block_bounds: smallest / largest key channel of every block of positions
  blocks      ct2x_attention_blocks: one token per entry over the blocks its bounds select

`run` computes the plain form in elementary torch operations, or - with `own` - makes the calls of
the C ABI. `exact` restates the definitions in float64, entry by entry.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_TYPE_IDS = {"f32": 0, "f16": 4, "bf16": 5}  # enum ct2x_dtype


# ---- cases ---------------------------------------------------------------------------------------


def listed():
    return [
        # five drafted tokens on a short sentence of the base Transformer (8 heads of 64): latency
        dict(name="tree_short_f32", op="tree", dtype="f32", batch=1, tokens=5, heads=8, heads_kv=8,
             dhead=64, length=150),
        # a server's ordinary verify step: 16 ragged conversations, 26 nodes, grouped heads
        dict(name="tree_batch_bf16", op="tree", dtype="bf16", batch=16, tokens=26, heads=32, heads_kv=8,
             dhead=128, length=2047),
        # long documents and wide trees: the most arithmetic of all cases
        dict(name="tree_long_bf16", op="tree", dtype="bf16", batch=4, tokens=64, heads=32, heads_kv=8,
             dhead=128, length=32000),
        # an odd head width, an odd group and odd lengths
        dict(name="tree_odd_f16", op="tree", dtype="f16", batch=3, tokens=17, heads=20, heads_kv=4,
             dhead=80, length=1501),
        # a decode step of the base Transformer that keeps weights: latency
        dict(name="accumulate_short_f32", op="accumulate", dtype="f32", batch=4, heads=8, heads_kv=8,
             dhead=64, length=333),
        # a decode step of a full server
        dict(name="accumulate_long_bf16", op="accumulate", dtype="bf16", batch=32, heads=32, heads_kv=8,
             dhead=128, length=8191),
        # a short chat that outgrew its budget
        dict(name="evict_short_f32", op="evict", dtype="f32", batch=2, heads_kv=8, dhead=64, length=500,
             budget=256, recent=64),
        # prompts of 16 k positions cut to a quarter after they were read
        dict(name="evict_prompt_bf16", op="evict", dtype="bf16", batch=8, heads_kv=8, dhead=128,
             length=16384, budget=4096, recent=512),
        # one token was appended to each of 32 entries: one block each
        dict(name="bounds_step_bf16", op="bounds", dtype="bf16", batch=32, heads_kv=8, dhead=128,
             length=8191, new=1, block=64),
        # a prompt was read: every block
        dict(name="bounds_prompt_f16", op="bounds", dtype="f16", batch=4, heads_kv=8, dhead=128,
             length=32768, new=32768, block=64),
        # small heads, small blocks
        dict(name="blocks_short_f32", op="blocks", dtype="f32", batch=2, heads=8, heads_kv=8, dhead=64,
             length=4100, block=32, top=24, sink=1, local=2),
        # a sixteenth of 64 k positions read per step
        dict(name="blocks_long_bf16", op="blocks", dtype="bf16", batch=8, heads=32, heads_kv=8,
             dhead=128, length=65536, block=64, top=64, sink=1, local=2),
    ]


def _between(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("tree", "tree", "accumulate", "evict", "bounds", "blocks"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    dhead = rng.choice((32, 64, 80, 96, 128, 128))
    heads_kv = rng.choice((1, 2, 4, 5, 8, 16))
    heads = heads_kv * rng.choice((1, 2, 4, 5, 8) if heads_kv <= 8 else (1, 2, 4))
    batch = _between(rng, 1, 32)
    element = 4 if dtype == "f32" else 2
    row = batch * heads_kv * dhead * element
    case = dict(op=op, dtype=dtype, batch=batch, heads_kv=heads_kv, dhead=dhead)
    # at most 0.4 GB of keys per cache, so that no drawn case costs more than the largest listed one
    longest = max(64, min(65536, 400_000_000 // row))
    if op == "tree":
        tokens = _between(rng, 1, 96)
        longest = max(64, min(longest, 60_000_000_000 // (4 * dhead * heads * tokens * batch)))
        if dtype == "f32":
            longest = max(64, longest // 4)
        case.update(heads=heads, tokens=tokens, length=_between(rng, 40, longest))
    elif op == "accumulate":
        case.update(heads=heads, length=_between(rng, 1, longest))
    elif op == "evict":
        length = _between(rng, 40, longest)
        budget = _between(rng, 16, max(17, length))
        case.update(length=length, budget=budget, recent=rng.randint(0, budget))
    elif op == "bounds":
        length = _between(rng, 40, longest)
        case.update(length=length, new=rng.choice((1, _between(rng, 1, length), length)),
                    block=rng.choice((16, 32, 48, 64, 128)))
    else:
        sink, local = rng.randint(0, 2), rng.randint(1, 3)
        case.update(heads=heads, length=_between(rng, 100, longest), block=rng.choice((16, 32, 48, 64, 128)),
                    top=sink + local + _between(rng, 1, 80), sink=sink, local=local)
    return case


def _lengths(case):
    """Ragged lengths: the longest first, down to about a quarter, odd ones among them."""
    n, b = case["length"], case["batch"]
    return [max(1, n - (3 * n * i) // (4 * b) - (i % 3)) if i else n for i in range(b)]


def _t_max(case):
    """The cache's room: a little more than the longest entry and its drafted tokens."""
    return case["length"] + case.get("tokens", 0) + 7


def _blocks_of(case):
    return -(-_t_max(case) // case["block"])


# ---- inputs --------------------------------------------------------------------------------------


def _cache(case, gen, spread):
    shape = (case["batch"], case["heads_kv"], _t_max(case), case["dhead"])
    x = torch.empty(shape, dtype=_DTYPES[case["dtype"]], device="cuda").normal_(generator=gen)
    if spread:  # keys have channels that stand out by an offset of their own
        offset = torch.randn((1, shape[1], 1, shape[3]), device="cuda", generator=gen)
        x += offset.to(x.dtype)
    return x


def _ancestors(case, gen):
    """mask[b, i, word]: bit j of the words says that drafted token i descends from token j (or is it)."""
    b, t = case["batch"], case["tokens"]
    # token i hangs under the last committed token or under one of the tokens before it
    parent = (torch.rand((b, t), device="cuda", generator=gen) * (torch.arange(t, device="cuda") + 1)).long() - 1
    seen = torch.eye(t, dtype=torch.bool, device="cuda").repeat(b, 1, 1)
    rows = torch.arange(b, device="cuda")
    for i in range(1, t):
        p = parent[:, i]
        seen[:, i] |= seen[rows, p.clamp(min=0)] & (p >= 0)[:, None]
    return _words(seen)


def _words(seen):
    b, t, _ = seen.shape
    n = -(-t // 64)
    bits = torch.zeros((b, t, n * 64), dtype=torch.int64, device=seen.device)
    bits[:, :, :t] = seen.long()
    return (bits.reshape(b, t, n, 64) << torch.arange(64, device=seen.device)).sum(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b, hkv, d = case["batch"], case["heads_kv"], case["dhead"]
    s = dict(case=case, scale=1.0 / math.sqrt(d), t_max=_t_max(case))
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    s["k"] = _cache(case, gen, True)
    if case["op"] != "bounds":
        s["v"] = _cache(case, gen, False)
    if case["op"] in ("tree", "accumulate", "blocks"):
        rows = (b, case["tokens"]) if case["op"] == "tree" else (b,)
        s["q"] = torch.randn(rows + (case["heads"], d), device="cuda", generator=gen) * 1.5
        s["out"] = torch.empty_like(s["q"])
    if case["op"] == "tree":
        s["mask"] = _ancestors(case, gen)
    if case["op"] in ("accumulate", "evict"):
        # most positions were hardly looked at, a few carry most of the weight, some none at all
        w = torch.empty((b, hkv, s["t_max"]), device="cuda").exponential_(generator=gen).pow_(4)
        w[torch.rand(w.shape, device="cuda", generator=gen) < 0.05] = 0
        s["weights"] = w
    if case["op"] == "evict":
        room = case["budget"]
        s["k_out"] = torch.zeros((b, hkv, room, d), dtype=s["k"].dtype, device="cuda")
        s["v_out"] = torch.zeros_like(s["k_out"])
        s["weights_out"] = torch.zeros((b, hkv, room), device="cuda")
        s["positions"] = torch.empty((b, hkv, room), dtype=torch.int32, device="cuda")
        s["lengths_out"] = torch.empty((b,), dtype=torch.int32, device="cuda")
    if case["op"] == "bounds":
        s["bounds"] = torch.zeros((b, hkv, _blocks_of(case), 2, d), dtype=s["k"].dtype, device="cuda")
        s["first"] = (s["lengths"] - case["new"]).clamp(min=0)
    if case["op"] == "blocks":
        s["bounds"] = _all_bounds(s["k"], s["lengths"], case["block"])
        s["selected"] = torch.empty((b, hkv, case["top"]), dtype=torch.int32, device="cuda")
    if case["op"] in ("tree", "accumulate", "evict", "blocks"):
        # the workspace of a serving loop: as large as any call of these sizes asks for
        s["scratch"] = torch.empty(_scratch_bytes(case), dtype=torch.uint8, device="cuda")
    return s


def _scratch_bytes(case):
    rows = case["batch"] * case.get("tokens", 1) * case.get("heads", case["heads_kv"])
    partials = (rows * 64 + 131072) * (case["dhead"] + 4) * 4
    scores = case["batch"] * case.get("heads", case["heads_kv"]) * (_t_max(case) + 64) * 8
    return partials + scores + (1 << 20)


def _all_bounds(k, lengths, block):
    b, hkv, t, d = k.shape
    n = -(-t // block)
    out = torch.empty((b, hkv, n, 2, d), dtype=k.dtype, device=k.device)
    full = t // block
    cut = k[:, :, :full * block].reshape(b, hkv, full, block, d)
    out[:, :, :full, 0] = cut.amin(3)
    out[:, :, :full, 1] = cut.amax(3)
    last = ((lengths.long() - 1) // block).clamp(min=0)  # the block that an entry's last position lies in
    at = last[:, None] * block + torch.arange(block, device=k.device)
    at = torch.minimum(at, (lengths.long() - 1)[:, None])
    rows = k[torch.arange(b, device=k.device)[:, None], :, at]  # [b, block, hkv, d]
    entry = torch.arange(b, device=k.device)
    out[entry, :, last, 0] = rows.amin(1)
    out[entry, :, last, 1] = rows.amax(1)
    return out


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    return (_OWN if own else _PLAIN)[op](state)


def _softmax_rows(scores, visible):
    """exp(x - max) over the visible columns, normalised; a row that sees nothing is all zero."""
    scores = torch.where(visible, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_tree(s):
    c, t = s["case"], s["case"]["tokens"]
    b, hkv, d = c["batch"], c["heads_kv"], c["dhead"]
    group = c["heads"] // hkv
    n = int(c["length"]) + t
    q = s["q"].reshape(b, t, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, t * group, d) * s["scale"]
    k, v = s["k"][:, :, :n].float(), s["v"][:, :, :n].float()
    position = torch.arange(n, device=q.device)
    behind = position - s["lengths"][:, None]  # [b, n]: which drafted token stands there
    word = (behind.clamp(min=0) // 64).clamp(max=s["mask"].shape[2] - 1)
    bits = torch.gather(s["mask"], 2, word[:, None].expand(b, t, n)) >> (behind.clamp(min=0) % 64)[:, None]
    visible = (behind < 0)[:, None] | (((bits & 1) == 1) & (behind >= 0)[:, None] & (behind < t)[:, None])
    visible = visible[:, None, :, None].expand(b, hkv, t, group, n).reshape(b, hkv, t * group, n)
    p = _softmax_rows(torch.matmul(q, k.transpose(2, 3).contiguous()), visible)
    out = torch.matmul(p, v).reshape(b, hkv, t, group, d)
    return out.permute(0, 2, 1, 3, 4).reshape(b, t, c["heads"], d)


def _plain_accumulate(s):
    c = s["case"]
    b, hkv, d, n = c["batch"], c["heads_kv"], c["dhead"], c["length"]
    q = s["q"].reshape(b, hkv, -1, d) * s["scale"]
    k, v = s["k"][:, :, :n].float(), s["v"][:, :, :n].float()
    visible = (torch.arange(n, device=q.device) < s["lengths"][:, None])[:, None, None]
    p = _softmax_rows(torch.matmul(q, k.transpose(2, 3).contiguous()), visible)
    s["weights"][:, :, :n] += p.sum(2)
    return [torch.matmul(p, v).reshape(b, c["heads"], d), s["weights"]]


def _plain_evict(s):
    c = s["case"]
    b, hkv, room = c["batch"], c["heads_kv"], c["budget"]
    n, t = s["lengths"].long(), s["t_max"]
    position = torch.arange(t, device=n.device)
    valid = (position < n[:, None])[:, None]
    newest = (position >= (n - c["recent"])[:, None])[:, None] & valid
    # the heaviest first, equal ones by position; the newest before all, nothing behind the end
    order = torch.where(newest, math.inf, torch.where(valid, s["weights"], -math.inf))
    chosen = torch.sort(order, dim=2, descending=True, stable=True).indices[:, :, :room]
    kept = torch.minimum(n, torch.full_like(n, room))
    filled = (torch.arange(chosen.shape[2], device=n.device) < kept[:, None])[:, None].expand(chosen.shape)
    chosen = torch.sort(torch.where(filled, chosen, t), dim=2).values
    if chosen.shape[2] < room:
        chosen = torch.nn.functional.pad(chosen, (0, room - chosen.shape[2]), value=t)
        filled = torch.nn.functional.pad(filled, (0, room - filled.shape[2]), value=False)
    at = chosen.clamp(max=t - 1)
    rows = at[..., None].expand(b, hkv, room, c["dhead"])
    zero = torch.zeros((), dtype=s["k"].dtype, device=n.device)
    return [torch.where(filled[..., None], torch.gather(s["k"], 2, rows), zero),
            torch.where(filled[..., None], torch.gather(s["v"], 2, rows), zero),
            torch.where(filled, torch.gather(s["weights"], 2, at), 0.0),
            torch.where(filled, chosen, -1).int(),
            kept.int()]


def _plain_bounds(s):
    c, k, block = s["case"], s["k"], s["case"]["block"]
    b, t = c["batch"], s["t_max"]
    touched = min(_blocks_of(c), (c["new"] + block - 2) // block + 1)
    n = s["lengths"].long()
    j = (s["first"].long() // block)[:, None] + torch.arange(touched, device=k.device)  # [b, touched]
    real = j * block < n[:, None]
    at = (j[..., None] * block + torch.arange(block, device=k.device)).reshape(b, -1)
    inside = (at < n[:, None])[:, None, :, None]
    rows = torch.gather(k, 2, at.clamp(max=t - 1)[:, None, :, None].expand(b, k.shape[1], at.shape[1], k.shape[3]))
    rows = rows.float()
    shape = (b, k.shape[1], touched, block, k.shape[3])
    low = torch.where(inside, rows, math.inf).reshape(shape).amin(3)
    high = torch.where(inside, rows, -math.inf).reshape(shape).amax(3)
    entry, number = torch.nonzero(real, as_tuple=True)
    s["bounds"][entry, :, j[entry, number], 0] = low[entry, :, number].to(k.dtype)
    s["bounds"][entry, :, j[entry, number], 1] = high[entry, :, number].to(k.dtype)
    return s["bounds"]


def _plain_blocks(s):
    c, block, top = s["case"], s["case"]["block"], s["case"]["top"]
    b, hkv, d, t = c["batch"], c["heads_kv"], c["dhead"], s["t_max"]
    q = s["q"].reshape(b, hkv, -1, d)
    n = s["lengths"].long()
    # the choice between blocks is made in 64 bits: q d >= 0 meets the largest key, q d < 0 the smallest
    low, high = s["bounds"][:, :, :, 0].double(), s["bounds"][:, :, :, 1].double()
    wide = q.double()
    score = torch.matmul(wide.clamp(min=0), high.transpose(2, 3)) + torch.matmul(wide.clamp(max=0), low.transpose(2, 3))
    score = score.amax(2)
    count = (n + block - 1) // block
    number = torch.arange(score.shape[2], device=q.device)
    valid = (number < count[:, None])[:, None]
    always = ((number < c["sink"]) | (number >= (count - c["local"])[:, None]))[:, None] & valid
    score = torch.where(always, math.inf, torch.where(valid, score, -math.inf))
    chosen = torch.sort(score, dim=2, descending=True, stable=True).indices[:, :, :top]
    filled = (torch.arange(chosen.shape[2], device=q.device) < count[:, None])[:, None].expand(chosen.shape)
    chosen = torch.sort(torch.where(filled, chosen, score.shape[2]), dim=2).values
    at = (chosen[..., None] * block + torch.arange(block, device=q.device)).reshape(b, hkv, -1)
    visible = (at < n[:, None, None])[:, :, None]
    rows = at.clamp(max=t - 1)[..., None].expand(b, hkv, at.shape[2], d)
    k, v = torch.gather(s["k"], 2, rows).float(), torch.gather(s["v"], 2, rows).float()
    p = _softmax_rows(torch.matmul(q * s["scale"], k.transpose(2, 3).contiguous()), visible)
    out = torch.matmul(p, v).reshape(b, c["heads"], d)
    chosen = torch.where(filled, chosen, -1).int()
    return [out, torch.nn.functional.pad(chosen, (0, top - chosen.shape[2]), value=-1)]


_PLAIN = {"tree": _plain_tree, "accumulate": _plain_accumulate, "evict": _plain_evict,
          "bounds": _plain_bounds, "blocks": _plain_blocks}


# ---- the framework's calls -----------------------------------------------------------------------


def _own_tree(s):
    from ctranslate2_amd import _lib
    c, p = s["case"], _lib.ptr
    _lib.check(_lib.lib().ct2x_attention_tree(
        p(s["q"]), p(s["k"]), p(s["v"]), _TYPE_IDS[c["dtype"]], p(s["lengths"]), 0, p(s["mask"]), c["batch"],
        c["tokens"], c["heads"], c["heads_kv"], c["dhead"], s["t_max"], s["scale"], p(s["out"]), p(s["scratch"]),
        s["scratch"].numel(), None))
    return s["out"]


def _own_accumulate(s):
    from ctranslate2_amd import _lib
    c, p = s["case"], _lib.ptr
    _lib.check(_lib.lib().ct2x_attention_accumulate(
        p(s["q"]), p(s["k"]), p(s["v"]), _TYPE_IDS[c["dtype"]], p(s["lengths"]), 0, c["batch"], c["heads"],
        c["heads_kv"], c["dhead"], s["t_max"], s["scale"], p(s["weights"]), p(s["out"]), p(s["scratch"]),
        s["scratch"].numel(), None))
    return [s["out"], s["weights"]]


def _own_evict(s):
    from ctranslate2_amd import _lib
    c, p = s["case"], _lib.ptr
    _lib.check(_lib.lib().ct2x_cache_evict(
        p(s["k"]), p(s["v"]), _TYPE_IDS[c["dtype"]], p(s["weights"]), p(s["lengths"]), 0, c["batch"], c["heads_kv"],
        c["dhead"], s["t_max"], c["budget"], c["recent"], c["budget"], p(s["k_out"]), p(s["v_out"]),
        p(s["weights_out"]), p(s["positions"]), p(s["lengths_out"]), p(s["scratch"]), s["scratch"].numel(), None))
    return [s["k_out"], s["v_out"], s["weights_out"], s["positions"], s["lengths_out"]]


def _own_bounds(s):
    from ctranslate2_amd import _lib
    c, p = s["case"], _lib.ptr
    _lib.check(_lib.lib().ct2x_cache_block_bounds(
        p(s["k"]), _TYPE_IDS[c["dtype"]], p(s["first"]), p(s["lengths"]), 0, c["batch"], c["heads_kv"], c["dhead"],
        s["t_max"], c["block"], p(s["bounds"]), None))
    return s["bounds"]


def _own_blocks(s):
    from ctranslate2_amd import _lib
    c, p = s["case"], _lib.ptr
    _lib.check(_lib.lib().ct2x_attention_blocks(
        p(s["q"]), p(s["k"]), p(s["v"]), _TYPE_IDS[c["dtype"]], p(s["bounds"]), p(s["lengths"]), 0, c["batch"],
        c["heads"], c["heads_kv"], c["dhead"], s["t_max"], c["block"], c["top"], c["sink"], c["local"], s["scale"],
        p(s["out"]), p(s["selected"]), p(s["scratch"]), s["scratch"].numel(), None))
    return [s["out"], s["selected"]]


_OWN = {"tree": _own_tree, "accumulate": _own_accumulate, "evict": _own_evict, "bounds": _own_bounds,
        "blocks": _own_blocks}


# ---- what a pass cannot do without ---------------------------------------------------------------


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    b, hkv, d, n = case["batch"], case["heads_kv"], case["dhead"], _lengths(case)
    heads = case.get("heads", 0)
    total = sum(n)
    if case["op"] == "tree":
        t = case["tokens"]
        return {"bytes": (total + b * t) * hkv * 2 * d * e + 2 * b * t * heads * d * 4,
                "flops": 4 * d * heads * t * (total + b * t)}
    if case["op"] == "accumulate":
        return {"bytes": total * hkv * (2 * d * e + 8) + 2 * b * heads * d * 4, "flops": 4 * d * heads * total}
    if case["op"] == "evict":
        kept = sum(min(x, case["budget"]) for x in n)
        return {"bytes": hkv * (4 * total + kept * (4 * d * e + 12)), "flops": hkv * total}
    block = case["block"]
    if case["op"] == "bounds":
        first = [max(0, x - case["new"]) // block for x in n]
        blocks = sum(-(-x // block) - f for x, f in zip(n, first))
        rows = sum(x - f * block for x, f in zip(n, first))
        return {"bytes": hkv * d * e * (rows + 2 * blocks), "flops": 2 * hkv * d * rows}
    blocks = sum(-(-x // block) for x in n)
    taken = sum(min(x, case["top"] * block) for x in n)
    return {"bytes": hkv * 2 * d * e * (blocks + taken) + 2 * b * heads * d * 4,
            "flops": heads * d * (2 * blocks + 4 * taken)}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "accumulate": _exact_accumulate, "evict": _exact_evict,
            "bounds": _exact_bounds, "blocks": _exact_blocks}[case["op"]](s, case)


def _exact_tree(s, c):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group, t = c["heads"] // c["heads_kv"], c["tokens"]
    bit = torch.arange(t, device="cuda")
    for b, n in enumerate(_lengths(c)):
        sees = torch.ones((t, n + t), dtype=torch.bool, device="cuda")
        sees[:, n:] = (s["mask"][b][:, bit // 64] >> (bit % 64)) & 1 == 1
        for h in range(c["heads"]):
            k, v = s["k"][b, h // group, :n + t].double(), s["v"][b, h // group, :n + t].double()
            x = s["q"][b, :, h].double() @ k.T / math.sqrt(c["dhead"])
            x[~sees] = -math.inf
            out[b, :, h] = torch.exp(x - torch.logsumexp(x, 1, keepdim=True)) @ v
    return out


def _exact_accumulate(s, c):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double()
    group = c["heads"] // c["heads_kv"]
    for b, n in enumerate(_lengths(c)):
        for h in range(c["heads"]):
            x = s["k"][b, h // group, :n].double() @ s["q"][b, h].double() / math.sqrt(c["dhead"])
            p = torch.exp(x - torch.logsumexp(x, 0))
            out[b, h] = p @ s["v"][b, h // group, :n].double()
            weights[b, h // group, :n] += p
    return [out, weights]


def _exact_evict(s, c):
    k, v, w = s["k_out"].double(), s["v_out"].double(), s["weights_out"].double()
    where = torch.full(w.shape, -1, dtype=torch.int32)
    for b, n in enumerate(_lengths(c)):
        old = max(0, n - c["recent"])
        heavy = min(max(0, c["budget"] - c["recent"]), old)
        if n <= c["budget"]:
            old = heavy = 0
        for h in range(c["heads_kv"]):
            x = s["weights"][b, h, :old].tolist()
            keep = sorted(sorted(range(old), key=lambda i: (-x[i], i))[:heavy]) + list(range(old, n))
            at = torch.tensor(keep, device="cuda")
            k[b, h, :len(keep)], v[b, h, :len(keep)] = s["k"][b, h, at].double(), s["v"][b, h, at].double()
            w[b, h, :len(keep)] = s["weights"][b, h, at].double()
            where[b, h, :len(keep)] = at.int().cpu()
    return [k, v, w, where, torch.tensor([min(n, c["budget"]) for n in _lengths(c)], dtype=torch.int32)]


def _exact_bounds(s, c):
    out = s["bounds"].double()
    for b, n in enumerate(_lengths(c)):
        for j in range(max(0, n - c["new"]) // c["block"], -(-n // c["block"])):
            rows = s["k"][b, :, j * c["block"]:min(n, (j + 1) * c["block"])].double()
            out[b, :, j, 0], out[b, :, j, 1] = rows.min(1).values, rows.max(1).values
    return out


def _exact_blocks(s, c):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    taken = torch.full((c["batch"], c["heads_kv"], c["top"]), -1, dtype=torch.int32)
    group = c["heads"] // c["heads_kv"]
    for b, n in enumerate(_lengths(c)):
        count = -(-n // c["block"])
        always = [j for j in range(count) if j < c["sink"] or j >= count - c["local"]]
        for g in range(c["heads_kv"]):
            q = s["q"][b, g * group:(g + 1) * group].double()
            low, high = s["bounds"][b, g, :count, 0].double(), s["bounds"][b, g, :count, 1].double()
            x = torch.stack([torch.maximum(one * low, one * high).sum(1) for one in q]).amax(0).tolist()
            others = sorted((j for j in range(count) if j not in always), key=lambda j: (-x[j], j))
            keep = sorted(always + others[:c["top"] - len(always)])
            taken[b, g, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
            at = torch.cat([torch.arange(j * c["block"], min(n, (j + 1) * c["block"])) for j in keep]).cuda()
            scores = q @ s["k"][b, g, at].double().T / math.sqrt(c["dhead"])
            p = torch.exp(scores - torch.logsumexp(scores, 1, keepdim=True))
            out[b, g * group:(g + 1) * group] = p @ s["v"][b, g, at].double()
    return [out, taken]
