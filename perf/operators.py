"""A serving step over a paged cache, as cases that can be timed and compared.

    listed()          the cases themselves
    draw(rng)         one more case from the same ranges
    prepare(case, s)  what a program has in hand before the call, on the GPU, made from seed s
    run(state)        one pass: the plain form in elementary torch operations, or, where `own` is true, the library's entry point
    work(case)        bytes and flops one pass cannot do without
    exact(case, s)    the same outputs in 64 bits

Four operators, in the order in which a step calls them:

    plan       yvex_b200_kv_plan          block tables, slot map, positions and ancestor masks from the requests' lengths
    append     yvex_b200_kv_append        the fresh tokens' keys and values into their pages
    attention  yvex_b200_attention_paged  the fresh tokens (one, a drafted chain or tree, a chunk of a prompt) over the pages
    logits     yvex_b200_logits_edit      penalties for repeated tokens, biases and grammar masks on the output head's rows

Queries, keys and values are N(0, 1) like the attention configuration's, logits N(0, 3); pages lie in random order, lengths are ragged.
"""
from __future__ import annotations

import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
TREE = 64                                   # most nodes of a drafted tree: its ancestor masks have 64 bits
VOCABULARY = 129280                         # rows of the benchmark's output head


def listed():
    return [
        # One token for each of 64 sessions: the bookkeeping of every decode step, all latency.
        dict(name="plan_decode", kind="plan", requests=64, fresh=1, longest=32768, page=64, tree=False),
        # Drafted trees for a full batch, captured for more rows than there are.
        dict(name="plan_trees", kind="plan", requests=512, fresh=64, longest=32768, page=16, tree=True),
        # The rows of a decode step as the projections leave them (f32) into a bf16 cache.
        dict(name="append_decode", kind="append", tokens=64, source="f32", dtype="bf16", kv_heads=8, dim=128, page=64, pages=4096),
        # The rows of a long prompt, already in the cache's type.
        dict(name="append_prompt", kind="append", tokens=16384, source="bf16", dtype="bf16", kv_heads=8, dim=128, page=64, pages=4096),
        # One session in a short conversation: the smallest attention call.
        dict(name="attend_1", kind="attention", requests=1, fresh=1, longest=1500, tree=False, dtype="bf16", q_heads=32, kv_heads=8, dim=128, page=64),
        # A decode step of 64 sessions of very different lengths.
        dict(name="attend_ragged", kind="attention", requests=64, fresh=1, longest=32768, tree=False, dtype="bf16", q_heads=32, kv_heads=8, dim=128,
             page=16),
        # A small drafted chain checked for a few sessions, odd group of query heads.
        dict(name="attend_chain_7", kind="attention", requests=5, fresh=7, longest=4001, tree=False, dtype="f16", q_heads=28, kv_heads=4, dim=64, page=48),
        # A drafted tree of one session: latency of verification.
        dict(name="attend_tree_1", kind="attention", requests=1, fresh=32, longest=8192, tree=True, dtype="bf16", q_heads=32, kv_heads=8, dim=128, page=64),
        # Full drafted trees for a batch of sessions at long contexts.
        dict(name="attend_trees", kind="attention", requests=16, fresh=64, longest=32768, tree=True, dtype="bf16", q_heads=32, kv_heads=8, dim=128,
             page=64),
        # Chunks of two prompts over what is cached of them: the largest, bound by the products.
        dict(name="attend_prompt", kind="attention", requests=2, fresh=4096, longest=8192, tree=False, dtype="bf16", q_heads=32, kv_heads=8, dim=128,
             page=64),
        # One session's logits.
        dict(name="logits_1", kind="logits", requests=1, fresh=1, tree=False, vocabulary=VOCABULARY, history=2000, biases=32, grammar=True, dtype="f32"),
        # A row for every node of a batch of drafted trees.
        dict(name="logits_trees", kind="logits", requests=16, fresh=32, tree=True, vocabulary=VOCABULARY, history=8000, biases=64, grammar=True, dtype="f32"),
    ]


# ---- sizes ------------------------------------------------------------------------------------------------------------

def _log(rng, lo, hi, step=1):
    """A size spread evenly over the logarithm of [lo, hi], a multiple of step."""
    v = lo * (hi / lo) ** rng.random()
    return int(min(hi, max(lo, round(v / step) * step)))


def draw(rng):
    kind = rng.choice(("plan", "append", "attention", "attention", "attention", "attention", "logits", "logits"))
    page = rng.choice((16, 16, 32, 48, 64, 64, 128, 256))
    if kind == "plan":
        tree = rng.random() < 0.5
        return dict(kind=kind, requests=_log(rng, 1, 512), fresh=_log(rng, 1, TREE), longest=_log(rng, 128, 32768), page=page, tree=tree)
    if kind == "append":
        return dict(kind=kind, tokens=_log(rng, 1, 16384), source=rng.choice(("f32", "bf16", "f16")), dtype=rng.choice(("bf16", "f16")),
                    kv_heads=rng.choice((1, 2, 4, 8)), dim=rng.choice((64, 128, 256)), page=page, pages=16384 // page + _log(rng, 1, 1000))
    if kind == "logits":
        while True:
            c = dict(kind=kind, requests=_log(rng, 1, 256), fresh=rng.choice((1, 1, _log(rng, 2, TREE))), tree=rng.random() < 0.5,
                     vocabulary=_log(rng, 1000, 151937), history=_log(rng, 1, 16000), biases=rng.choice((0, _log(rng, 1, 300))),
                     grammar=rng.random() < 0.7, dtype=rng.choice(("f32", "f32", "bf16", "f16")))
            if c["requests"] * c["fresh"] * c["vocabulary"] <= 512 * VOCABULARY and c["requests"] * c["history"] <= 200000:
                return c
    while True:
        form = rng.choice(("decode", "chain", "tree", "prompt"))
        kv = rng.choice((1, 2, 4, 8, 8, 16))
        c = dict(kind=kind, requests=_log(rng, 1, 4 if form == "prompt" else 64),
                 fresh={"decode": 1, "chain": _log(rng, 2, 16), "tree": _log(rng, 2, TREE), "prompt": _log(rng, 65, 4096)}[form],
                 longest=_log(rng, 100, 65536), tree=form == "tree", dtype=rng.choice(("bf16", "bf16", "f16")),
                 q_heads=kv * rng.choice((1, 2, 4, 4, 5, 7, 8, 16)), kv_heads=kv, dim=rng.choice((64, 128, 128, 256)), page=page)
        c["longest"] = max(c["longest"], c["fresh"])
        if (c["requests"] * kv * c["longest"] * c["dim"] <= 16 * 8 * 32768 * 128 and
                c["requests"] * c["q_heads"] * c["fresh"] * c["longest"] <= 16 * 32 * 64 * 32768 and
                c["requests"] * c["q_heads"] * c["fresh"] * c["longest"] * c["dim"] <= 2 * 32 * 4096 * 8192 * 128):
            return c


def _fresh(c, rng):
    """Fresh tokens of every request: the most, then half of that and more."""
    return [c["fresh"]] + [rng.randint(max(1, c["fresh"] // 2), c["fresh"]) for _ in range(c["requests"] - 1)]


def _lengths(c):
    """(cached, fresh) of every request: the longest and some short ones, in an order of their own; fixed by the case's sizes."""
    rng = random.Random("%d %d %d" % (c["requests"], c["fresh"], c["longest"]))
    fresh = _fresh(c, rng)
    total = [c["longest"]] + [max(f, int(c["longest"] * rng.random() ** 1.5)) for f in fresh[1:]]
    both = [(n - f, f) for n, f in zip(total, fresh)]
    rng.shuffle(both)
    return [a for a, _ in both], [b for _, b in both]


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed & 0x7fffffff)
    return gen


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _up(a, b):
    return -(-a // b)


def _prefix(n):
    return torch.cat([n.new_zeros(1), torch.cumsum(n, 0)])


def _parents(fresh, rows, gen):
    """A parent for every row, an index within its request below the row's own (-1: the row hangs on the cache)."""
    index = torch.arange(rows, device="cuda") - torch.repeat_interleave(_prefix(fresh)[:-1], fresh, output_size=rows)
    parent = (torch.rand(rows, device="cuda", generator=gen) * index).floor().long()
    return torch.where(index == 0, torch.full_like(parent, -1), parent).to(torch.int32)


def _closure(parents, offsets):
    """[requests, TREE, TREE] truth values: node i of a request's tree sees node j (itself and all its ancestors)."""
    requests, rows = offsets.numel() - 1, parents.numel()
    row = torch.arange(rows, device="cuda")
    request = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp(max=requests - 1)
    index, parent = row - offsets[request], parents.long()
    live = (row < offsets[-1]) & (parent >= 0)
    step = torch.eye(TREE, dtype=torch.float64, device="cuda").repeat(requests, 1, 1)
    step[request[live], index[live], parent[live]] = 1.0
    return torch.linalg.matrix_power(step, TREE) > 0


def _bits(sees):
    """Truth values [.., TREE] as the bits of one 64-bit number."""
    return (sees.long() << torch.arange(TREE, device="cuda")).sum(-1)


def _masks(parents, offsets):
    """The ancestor mask of every row (0 behind the last one)."""
    rows = parents.numel()
    row = torch.arange(rows, device="cuda")
    request = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp(max=offsets.numel() - 2)
    mask = _bits(_closure(parents, offsets))[request, (row - offsets[request]).clamp(max=TREE - 1)]
    return torch.where(row < offsets[-1], mask, torch.zeros_like(mask))


def prepare(case, seed):
    c, gen = case, _generator(seed)
    randn = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    s = dict(case=c)
    if c["kind"] == "append":
        slots = torch.randperm(c["pages"] * c["page"], device="cuda", generator=gen)[:c["tokens"]]
        s["slots"] = torch.where(torch.rand(c["tokens"], device="cuda", generator=gen) < 0.02, torch.full_like(slots, -1), slots)  # some rows are padding
        # keys and values as a projection leaves them: one row [k | v] a token
        s["rows"] = randn(c["tokens"], 2, c["kv_heads"], c["dim"]).to(DTYPES[c["source"]])
        s["k"], s["v"] = (torch.zeros((c["pages"], c["kv_heads"], c["page"], c["dim"]), dtype=DTYPES[c["dtype"]], device="cuda") for _ in range(2))
        return s
    if c["kind"] == "logits":
        rng = random.Random("%d %d %d" % (c["requests"], c["fresh"], c["history"]))
        fresh = _fresh(c, rng)
        history = [c["history"]] + [int(c["history"] * rng.random()) for _ in range(c["requests"] - 1)]
        s["fresh"], s["rows"] = _ints(fresh), sum(fresh)
        s["offsets"] = _prefix(s["fresh"].long())
        s["row_request"] = torch.repeat_interleave(torch.arange(c["requests"], device="cuda"), s["fresh"].long(), output_size=s["rows"]).to(torch.int32)
        s["ancestors"] = _masks(_parents(s["fresh"].long(), s["rows"], gen), s["offsets"]) if c["tree"] else None
        zipf = lambda n: (c["vocabulary"] ** torch.rand(n, device="cuda", generator=gen) - 1).long().clamp(max=c["vocabulary"] - 1).to(torch.int32)  # noqa: E731
        s["drafted"], s["history"] = zipf(s["rows"]), zipf(max(1, sum(history)))          # few words make up most of a text
        s["history_offsets"] = _prefix(_ints(history, torch.int64)).to(torch.int32)
        s["prompt"] = _ints([int(h * rng.random()) for h in history])
        uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(c["requests"], device="cuda", generator=gen)  # noqa: E731
        s["repetition"], s["presence"], s["frequency"] = uniform(1.0, 1.3), uniform(0.0, 1.0), uniform(0.0, 0.5)
        s["bias_tokens"] = s["bias_values"] = s["bias_offsets"] = None
        if c["biases"]:
            s["bias_tokens"] = torch.cat([torch.randperm(c["vocabulary"], device="cuda", generator=gen)[:c["biases"]] for _ in range(c["requests"])]).to(torch.int32)
            s["bias_values"] = 5.0 * randn(c["requests"] * c["biases"])
            s["bias_offsets"] = torch.arange(c["requests"] + 1, device="cuda", dtype=torch.int32) * c["biases"]
        words = _up(c["vocabulary"], 32)
        s["grammar"] = (torch.randint(-2**31, 2**31, (s["rows"], words), device="cuda", generator=gen, dtype=torch.int64).to(torch.int32)
                        if c["grammar"] else None)
        s["logits"] = (3.0 * randn(s["rows"], c["vocabulary"])).to(DTYPES[c["dtype"]])
        s["out"] = torch.empty_like(s["logits"])
        return s
    cached, fresh = _lengths(c)
    total = [a + b for a, b in zip(cached, fresh)]
    s["cached"], s["fresh"], s["rows"] = _ints(cached), _ints(fresh), sum(fresh)
    s["width"] = _up(c["longest"], c["page"])
    used = [_up(n, c["page"]) for n in total]
    pages = sum(used) + 7
    order = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
    s["table"] = torch.full((c["requests"], s["width"]), -1, dtype=torch.int32, device="cuda")
    column = torch.arange(s["width"], device="cuda")[None]
    held = [_up(n, c["page"]) for n in (cached if c["kind"] == "plan" else total)]
    first = _prefix(_ints(held, torch.int64))
    s["table"] = torch.where(column < _ints(held)[:, None], order[(first[:-1, None] + column).clamp(max=pages - 1)], s["table"]).contiguous()
    if c["kind"] == "plan":
        s["free"], s["pages"] = order[int(sum(held)):].contiguous(), pages
        s["capacity"] = c["requests"] * c["fresh"]                      # a graph is captured for the most rows there can be
        parents = _parents(s["fresh"].long(), s["rows"], gen)
        s["parents"] = torch.cat([parents, parents.new_full((s["capacity"] - s["rows"],), -1)]) if c["tree"] else None
        return s
    s["offsets"] = _prefix(s["fresh"].long())
    s["ancestors"] = _masks(_parents(s["fresh"].long(), s["rows"], gen), s["offsets"]) if c["tree"] else None
    kind = DTYPES[c["dtype"]]
    s["q"] = randn(s["rows"], c["q_heads"], c["dim"]).to(kind)
    s["k"], s["v"] = (torch.empty((pages, c["kv_heads"], c["page"], c["dim"]), dtype=kind, device="cuda").normal_(generator=gen) for _ in range(2))
    s["out"] = torch.empty_like(s["q"])
    return s


# ---- the library's calls ----------------------------------------------------------------------------------------------

def _handles(s):
    """What a program builds once for its buffers: the status word, the descriptions of cache and step, the workspace."""
    from yvex_b200 import lib
    c, h = s["case"], {}
    h["lib"], h["status"] = lib, lib.Status()
    if c["kind"] in ("append", "attention"):
        h["cache"] = lib.kv_cache_of(s["k"], s["v"])
    if c["kind"] == "plan":
        h["cache"] = lib.kv_geometry_of(s["pages"], c["page"])
        h["step"] = lib.kv_step_of(s["cached"], s["fresh"], s["table"], tokens=s["capacity"], longest_fresh=c["fresh"], longest=c["longest"],
                                   parents=s["parents"])
        h["used"] = torch.empty(1, dtype=torch.int32, device="cuda")
    if c["kind"] == "attention":
        h["step"] = lib.kv_step_of(s["cached"], s["fresh"], s["table"], tokens=s["rows"], longest_fresh=c["fresh"], longest=c["longest"],
                                   offsets=s["offsets"].to(torch.int32), ancestors=s["ancestors"], tree=c["tree"])
        h["workspace"] = lib.attention_paged_workspace(h["cache"], h["step"], c["q_heads"])
    if c["kind"] == "logits":
        h["policy"] = lib.logits_policy_of(c["vocabulary"], s["history"], s["history_offsets"], s["prompt"], s["repetition"], s["presence"], s["frequency"],
                                           s["bias_tokens"], s["bias_values"], s["bias_offsets"])
        h["drafts"] = lib.logits_drafts_of(s["drafted"], s["row_request"], s["offsets"].to(torch.int32), s["ancestors"], tree=c["tree"])
    return h


def _own(s):
    c = s["case"]
    if "handles" not in s:
        s["handles"] = _handles(s)
    h = s["handles"]
    lib = h["lib"]
    if c["kind"] == "plan":
        lib.kv_plan(h["cache"], h["step"], s["free"], h["status"], pages_used=h["used"])
        t = h["step"]
        out = dict(table=s["table"], offsets=t.offsets_tensor, slots=t.slots_tensor, positions=t.positions_tensor, row_request=t.row_request_tensor,
                   pages_used=h["used"])
        return dict(out, ancestors=t.ancestors_tensor) if c["tree"] else out
    if c["kind"] == "append":
        lib.kv_append(h["cache"], s["slots"], s["rows"][:, 0], s["rows"][:, 1], h["status"])
        return dict(k=s["k"], v=s["v"])
    if c["kind"] == "attention":
        return lib.attention_paged(h["cache"], h["step"], s["q"], c["dim"] ** -0.5, h["status"], workspace=h["workspace"], out=s["out"])
    return lib.logits_edit(h["policy"], h["drafts"], s["logits"], h["status"], grammar=s["grammar"], out=s["out"])


# ---- the plain forms --------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _own(state)
    return dict(plan=_plan, append=_append, attention=_attention, logits=_logits)[state["case"]["kind"]](state)


def _plan(s):
    c, page = s["case"], s["case"]["page"]
    cached, fresh = s["cached"].long(), s["fresh"].long()
    offsets = _prefix(fresh)
    held, most = (cached + page - 1) // page, (cached + fresh + page - 1) // page
    first = _prefix(most - held)
    column = torch.arange(s["width"], device="cuda")[None]
    taken = (first[:-1] - held)[:, None] + column
    s["table"].copy_(torch.where((column >= held[:, None]) & (column < most[:, None]), s["free"][taken.clamp(0, s["free"].numel() - 1)], s["table"]))
    row = torch.arange(s["capacity"], device="cuda")
    request = torch.searchsorted(offsets[1:].contiguous(), row, right=True).clamp(max=c["requests"] - 1)
    live, index = row < offsets[-1], row - offsets[request]
    at = (cached[request] + index).clamp(max=s["width"] * page - 1)
    slots = s["table"][request, at // page].long() * page + at % page
    out = dict(table=s["table"], offsets=offsets.to(torch.int32), slots=torch.where(live, slots, torch.full_like(slots, -1)),
               row_request=torch.where(live, request, torch.full_like(request, -1)).to(torch.int32), pages_used=first[-1:].to(torch.int32))
    if c["tree"]:
        sees = _closure(s["parents"], offsets)[request, index.clamp(max=TREE - 1)]
        out["ancestors"] = torch.where(live, _bits(sees), torch.zeros_like(row))
        index = sees.sum(-1) - 1
    out["positions"] = torch.where(live, cached[request] + index, torch.zeros_like(row)).to(torch.int32)
    return out


def _append(s):
    page = s["case"]["page"]
    live = s["slots"] >= 0
    slots, rows = s["slots"][live], s["rows"][live].to(s["k"].dtype)
    s["k"][slots // page, :, slots % page] = rows[:, 0]
    s["v"][slots // page, :, slots % page] = rows[:, 1]
    return dict(k=s["k"], v=s["v"])


def _attention(s):
    c, page = s["case"], s["case"]["page"]
    R, T, L, H, G, D = c["requests"], c["fresh"], s["width"] * c["page"], c["kv_heads"], c["q_heads"] // c["kv_heads"], c["dim"]
    cached, fresh, offsets = s["cached"].long(), s["fresh"].long(), s["offsets"]
    k, v = (s[n][s["table"].clamp(min=0).long()].transpose(1, 2).reshape(R, H, L, D).float() for n in ("k", "v"))
    node = torch.arange(T, device="cuda")
    row = (offsets[:-1, None] + node).clamp(max=s["rows"] - 1)                              # [R, T]
    key = torch.arange(L, device="cuda")[None, None] - cached[:, None, None]                # [R, 1, L]: index among the fresh tokens
    if c["tree"]:
        sees = (key < 0) | ((key < TREE) & ((s["ancestors"][row][:, :, None] >> key.clamp(0, TREE - 1)) & 1 == 1))
    else:
        sees = key <= node[None, :, None]
    sees = sees & (key < fresh[:, None, None])
    q = s["q"][row].float().reshape(R, T, H, G, D).permute(0, 2, 3, 1, 4).reshape(R, H, G * T, D)
    score = (q @ k.transpose(2, 3)).mul_(D ** -0.5).reshape(R, H, G, T, L)
    score = score.masked_fill_(~sees[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = (weight.reshape(R, H, G * T, L) @ v).reshape(R, H, G, T, D) / torch.where(total == 0, torch.ones_like(total), total)
    out = out.permute(0, 3, 1, 2, 4).reshape(R, T, H * G, D)
    return out[node[None] < fresh[:, None]].to(s["q"].dtype)


def _edits(s, dtype):
    """What the edits go by, per row and word: seen at all, times generated, bias (0 without)."""
    c, R, V = s["case"], s["case"]["requests"], s["case"]["vocabulary"]
    history, first, prompt = s["history"].long(), s["history_offsets"].long(), s["prompt"].long()
    at = torch.arange(history.numel(), device="cuda")
    request = torch.searchsorted(first[1:].contiguous(), at, right=True).clamp(max=R - 1)
    live = at < first[-1]
    where = torch.where(live, request * V + history, torch.zeros_like(at))
    seen = torch.zeros(R * V, dtype=torch.int32, device="cuda").scatter_add_(0, where, live.to(torch.int32)).reshape(R, V)
    made = torch.zeros(R * V, dtype=torch.int32, device="cuda").scatter_add_(0, where, (live & (at - first[request] >= prompt[request])).to(torch.int32)).reshape(R, V)
    of, offsets = s["row_request"].long(), s["offsets"]
    row, node = torch.arange(s["rows"], device="cuda"), torch.arange(c["fresh"], device="cuda")
    index = row - offsets[of]
    on = (s["ancestors"][:, None] >> node) & 1 == 1 if c["tree"] else node <= index[:, None]     # [rows, fresh]: the drafted words of the row's path
    word = s["drafted"].long()[(offsets[of][:, None] + node).clamp(max=s["rows"] - 1)]
    path = torch.zeros((s["rows"], V), dtype=torch.int32, device="cuda").scatter_add_(1, word, on.to(torch.int32))
    bias = torch.zeros((R, V), dtype=dtype, device="cuda")
    if c["biases"]:
        bias.scatter_(1, s["bias_tokens"].long().reshape(R, -1), s["bias_values"].to(dtype).reshape(R, -1))
    return of, seen[of] + path > 0, made[of] + path, bias[of]


def _edited(s, dtype):
    c = s["case"]
    of, seen, count, bias = _edits(s, dtype)
    x = s["logits"].to(dtype)
    repetition, presence, frequency = (s[n].to(dtype)[of][:, None] for n in ("repetition", "presence", "frequency"))
    x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
    x = x - frequency * count - presence * (count > 0) + bias
    if c["grammar"]:
        word = torch.arange(c["vocabulary"], device="cuda")
        x = x.masked_fill((s["grammar"][:, word // 32] >> (word % 32)) & 1 == 0, float("-inf"))
    return x


def _logits(s):
    return _edited(s, torch.float32).to(s["logits"].dtype)


# ---- what a pass needs ------------------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "append":
        values = 2 * c["tokens"] * c["kv_heads"] * c["dim"]
        return {"bytes": 8 * c["tokens"] + values * (2 + (4 if c["source"] == "f32" else 2)), "flops": 0}
    if c["kind"] == "logits":
        rows = sum(_fresh(c, random.Random("%d %d %d" % (c["requests"], c["fresh"], c["history"]))))
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": rows * c["vocabulary"] * (2 * size + (0.125 if c["grammar"] else 0)) + 2 * c["requests"] * c["history"] + 8 * c["requests"] * c["biases"],
                "flops": 4 * rows * c["vocabulary"]}
    cached, fresh = _lengths(c)
    if c["kind"] == "plan":
        rows = c["requests"] * c["fresh"]
        pages = sum(_up(a + b, c["page"]) - _up(a, c["page"]) for a, b in zip(cached, fresh))
        return {"bytes": 12 * c["requests"] + 16 * rows + 8 * pages + (8 * rows + 4 * sum(fresh) if c["tree"] else 0), "flops": 0}
    seen = sum(f * a + (f if c["tree"] else f * (f + 1) / 2) for a, f in zip(cached, fresh))       # (token, key) pairs
    keys = sum(a + f for a, f in zip(cached, fresh))
    return {"bytes": 4 * c["dim"] * (c["kv_heads"] * keys + c["q_heads"] * sum(fresh)), "flops": 4 * c["dim"] * c["q_heads"] * seen}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "plan":
        return None                                                      # whole numbers
    if c["kind"] == "append":
        out = {}
        for side, name in enumerate("kv"):
            rows = torch.zeros((c["pages"] * c["page"], c["kv_heads"], c["dim"]), dtype=torch.float64, device="cuda")
            rows[s["slots"][s["slots"] >= 0]] = s["rows"][s["slots"] >= 0, side].double()
            out[name] = rows.reshape(c["pages"], c["page"], c["kv_heads"], c["dim"]).transpose(1, 2)
        return out
    if c["kind"] == "logits":
        rows = s["logits"].double()
        of = s["row_request"].tolist()
        first, begin = s["history_offsets"].tolist(), s["offsets"].tolist()
        prompt = s["prompt"].tolist()
        history, drafted = s["history"].long(), s["drafted"].long()
        for t, r in enumerate(of):
            i = t - begin[r]
            path = ([j for j in range(c["fresh"]) if int(s["ancestors"][t]) >> j & 1] if c["tree"] else list(range(i + 1)))
            words = torch.cat([history[first[r]:first[r + 1]], drafted[[begin[r] + j for j in path]]])
            seen = torch.bincount(words, minlength=c["vocabulary"]) > 0
            count = torch.bincount(words[min(prompt[r], first[r + 1] - first[r]):], minlength=c["vocabulary"]).double()
            x, repetition = rows[t], s["repetition"][r].double()
            x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
            x = x - s["frequency"][r].double() * count - s["presence"][r].double() * (count > 0)
            if c["biases"]:
                a, b = int(s["bias_offsets"][r]), int(s["bias_offsets"][r + 1])
                x[s["bias_tokens"][a:b].long()] += s["bias_values"][a:b].double()
            rows[t] = x
        if c["grammar"]:
            bits = (s["grammar"][:, :, None] >> torch.arange(32, device="cuda")) & 1
            rows[bits.reshape(s["rows"], -1)[:, :c["vocabulary"]] == 0] = float("-inf")
        return rows
    page, G, D = c["page"], c["q_heads"] // c["kv_heads"], c["dim"]
    out = torch.zeros((s["rows"], c["q_heads"], D), dtype=torch.float64, device="cuda")
    cached, fresh, begin = s["cached"].tolist(), s["fresh"].tolist(), s["offsets"].tolist()
    for r in range(c["requests"]):
        n, f, b = cached[r] + fresh[r], fresh[r], begin[r]
        at = torch.arange(n, device="cuda")
        held = s["table"][r].long()[at // page]
        sees = torch.ones((f, n), dtype=torch.bool, device="cuda")
        if c["tree"]:
            sees[:, cached[r]:] = (s["ancestors"][b:b + f, None] >> torch.arange(f, device="cuda")) & 1 == 1
        else:
            sees[:, cached[r]:] = torch.ones((f, f), dtype=torch.bool, device="cuda").tril()
        for h in range(c["kv_heads"]):
            k, v = (s[x][held, h, at % page].double() for x in ("k", "v"))
            q = s["q"][b:b + f, h * G:(h + 1) * G].double().reshape(f * G, D)
            score = (q @ k.T * D ** -0.5).reshape(f, G, n).masked_fill(~sees[:, None], float("-inf"))
            out[b:b + f, h * G:(h + 1) * G] = (torch.softmax(score, -1).reshape(f * G, n) @ v).reshape(f, G, D)
    return out
