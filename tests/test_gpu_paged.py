"""A serving step over a paged cache on a B200: plan, append, attention and logit edits against plain restatements in 64 bits."""
import numpy as np
import pytest

import paged_oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from yvex_b200 import lib
    return lib


def ints(values, dtype=None):
    import torch
    return torch.tensor(values, dtype=dtype or torch.int32, device="cuda")


def up(a, b):
    return -(-a // b)


class Step:
    """Lengths, a page pool in random order and the table of what is cached; `plan()` runs the library, `want` is the restatement."""

    def __init__(self, L, cached, fresh, page, seed=0, tree=None, extra_tokens=0, extra_pages=5, extra_width=1):
        import torch
        rng = np.random.default_rng(seed)
        self.L, self.cached, self.fresh, self.page, self.rng = L, list(cached), list(fresh), page, rng
        self.tokens = max(1, sum(fresh) + extra_tokens)
        self.width = max(1, max(up(c + f, page) for c, f in zip(cached, fresh)) + extra_width)
        held = [up(c, page) for c in cached]
        total = sum(up(c + f, page) for c, f in zip(cached, fresh))
        self.pages = total + extra_pages
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = rng.integers(-5, 1 << 30, (len(cached), self.width)).astype(np.int32)       # rubbish where nothing is held
        at = 0
        for r, h in enumerate(held):
            self.table[r, :h] = order[at:at + h]
            at += h
        self.free = order[at:].copy()
        self.parents = O.parents_of(rng, fresh, tree) if tree else None
        self.table_dev, self.free_dev = ints(self.table), ints(self.free)
        padded = None if self.parents is None else ints(self.parents + [7] * (self.tokens - sum(fresh)))
        self.cached_dev, self.fresh_dev = ints(self.cached), ints(self.fresh)
        self.step = L.kv_step_of(self.cached_dev, self.fresh_dev, self.table_dev, self.tokens, max(1, max(fresh)),
                                 max(1, max(c + f for c, f in zip(cached, fresh))), parents=padded)
        self.status = L.Status()
        self.want = O.plan(self.cached, self.fresh, self.table, self.free, page, self.tokens, self.parents)
        self.torch = torch

    def plan(self):
        return self.L.kv_plan(self.L.kv_geometry_of(self.pages, self.page), self.step, self.free_dev, self.status)

    def check_plan(self, used):
        s, w = self.step, self.want
        assert s.offsets_tensor.tolist() == w["offsets"]
        assert s.slots_tensor.tolist() == w["slots"]
        assert s.positions_tensor.tolist() == w["positions"]
        assert s.row_request_tensor.tolist() == w["row_request"]
        if self.parents is not None:
            assert s.ancestors_tensor.tolist() == [O.signed(m) for m in w["ancestors"]]
        assert used.tolist() == [w["taken"]]
        assert np.array_equal(self.table_dev.cpu().numpy(), self.table)

    def masks(self):
        return self.want["ancestors"] if self.parents is not None else None


LENGTHS = [([0], [1]), ([15], [1]), ([16], [1]), ([0, 0, 0], [0, 5, 0]), ([5, 100, 0, 31], [1, 17, 64, 0]), ([0], [700]), ([37, 9], [515, 1000])]


@pytest.mark.parametrize("page", [16, 48, 256])
@pytest.mark.parametrize("tree", [None, "random", "chain", "star"])
@pytest.mark.parametrize("which", range(len(LENGTHS)))
def test_plan(L, which, tree, page):
    cached, fresh = LENGTHS[which]
    if tree and max(fresh) > 64:
        pytest.skip("more nodes than a tree has")
    s = Step(L, cached, fresh, page, seed=which, tree=tree, extra_tokens=3)
    used = s.plan()
    assert s.status.read() == 0
    s.check_plan(used)
    used = s.plan()                                              # the same plan again: nothing it reads has changed
    assert s.status.read() == 0
    s.check_plan(used)


@pytest.mark.parametrize("requests", [511, 512, 513, 1300])
@pytest.mark.parametrize("tree", [None, "random"])
def test_plan_many_requests(L, requests, tree):
    """More requests than a CTA scans at a time, many without fresh tokens, rows of one CTA in requests of another's chunk."""
    rng = np.random.default_rng(requests)
    cached = rng.integers(0, 300, requests).tolist()
    fresh = (rng.integers(0, 13, requests) * (rng.random(requests) < 0.6)).tolist()
    s = Step(L, cached, fresh, 16, seed=requests, tree=tree, extra_tokens=40)
    used = s.plan()
    assert s.status.read() == 0
    s.check_plan(used)


def test_plan_without_fresh_tokens(L):
    s = Step(L, [3, 0], [0, 0], 16, extra_tokens=2)
    used = s.plan()
    assert s.status.read() == 0
    s.check_plan(used)


def test_plan_reports_what_it_cannot_plan(L):
    """Bad inputs set status 2; the rows that are in order are planned all the same."""
    # too few free pages: the second request's rows past its held page get no slot
    s = Step(L, [10, 10], [10, 10], 16)
    s.free_dev = s.free_dev[:1].contiguous()
    s.plan()
    assert s.status.read() == 2
    want = s.want["slots"]
    assert s.step.slots_tensor.tolist() == want[:16] + [-1] * 4
    # a table that is too narrow
    s = Step(L, [10], [10], 16)
    narrow = L.kv_step_of(s.cached_dev, s.fresh_dev, ints([[2]]), 10, 10, 20)
    L.kv_plan(L.kv_geometry_of(s.pages, 16), narrow, s.free_dev, s.status)
    assert s.status.read() == 2 and narrow.slots_tensor.tolist() == [2 * 16 + 10 + i for i in range(6)] + [-1] * 4
    # a page outside the cache, in the table and among the free ones
    for bad in (-1, 1 << 20):
        s = Step(L, [10], [3], 16)
        s.table_dev[0, 0] = bad
        s.plan()
        assert s.status.read() == 2 and s.step.slots_tensor.tolist() == [-1] * 3
        s = Step(L, [16], [3], 16)
        s.free_dev[0] = bad
        s.plan()
        assert s.status.read() == 2 and s.step.slots_tensor.tolist() == [-1] * 3
        assert int(s.table_dev[0, 1]) not in (bad,)
    # negative lengths count as nothing, lengths above their bounds are reported
    s = Step(L, [4, 4], [2, 2], 16)
    s.fresh_dev[0] = -3
    s.plan()
    assert s.status.read() == 2 and s.step.offsets_tensor.tolist() == [0, 0, 2] and s.step.row_request_tensor.tolist() == [1, 1, -1, -1]
    s = Step(L, [4, 4], [2, 2], 16)
    s.fresh_dev[1] = 3
    s.plan()
    assert s.status.read() == 2 and s.step.offsets_tensor.tolist() == [0, 2, 5]
    # a parent that is not before its child counts as none
    s = Step(L, [4], [4], 16, tree="chain")
    parents = ints([-1, 1, -7, 0])
    step = L.kv_step_of(s.cached_dev, s.fresh_dev, s.table_dev, 4, 4, 8, parents=parents)
    L.kv_plan(L.kv_geometry_of(s.pages, 16), step, s.free_dev, s.status)
    assert s.status.read() == 2 and step.ancestors_tensor.tolist() == [1, 2, 4, 9]


@pytest.mark.parametrize("source", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("tokens,heads,dim,page,packed", [(1, 1, 64, 16, True), (7, 2, 128, 16, False), (65, 3, 256, 48, False), (300, 8, 128, 64, False),
                                                          (33, 1, 128, 400, True)])
def test_append(L, source, dtype, tokens, heads, dim, page, packed):
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(tokens)
    pages = up(tokens, page) + 3
    k, v = (torch.randn((pages, heads, page, dim), device="cuda", generator=gen).to(getattr(torch, dtype)) for _ in range(2))
    want = [k.clone(), v.clone()]
    slots = torch.randperm(pages * page, device="cuda", generator=gen)[:tokens]
    slots[torch.rand(tokens, device="cuda", generator=gen) < 0.2] = -1
    rows = (100 * torch.randn((tokens, 2, heads, dim), device="cuda", generator=gen)).to(getattr(torch, source))
    rk, rv = (rows[:, i].contiguous() if packed else rows[:, i] for i in range(2))
    st = L.Status()
    L.kv_append(L.kv_cache_of(k, v), slots, rk, rv, st)
    assert st.read() == 0
    for t, slot in enumerate(slots.tolist()):
        if slot >= 0:
            want[0][slot // page, :, slot % page] = rows[t, 0].to(k.dtype)
            want[1][slot // page, :, slot % page] = rows[t, 1].to(k.dtype)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_append_reports_slots_past_the_cache_and_values_that_are_not_finite(L):
    import torch
    k, v = (torch.zeros((4, 2, 16, 64), dtype=torch.float16, device="cuda") for _ in range(2))
    rows = torch.ones((3, 2, 64), device="cuda")
    st = L.Status()
    L.kv_append(L.kv_cache_of(k, v), ints([3, 64, 1 << 40], torch.int64), rows, rows, st)
    assert st.read() == 2 and float(k.sum()) == 128 and float(v.sum()) == 128 and float(k[0, :, 3].sum()) == 128
    for bad in (1e6, float("nan"), float("inf")):
        st.reset()
        rows[1, 1, 63] = bad
        L.kv_append(L.kv_cache_of(k, v), ints([0, 1, 2], torch.int64), rows, rows, st)
        assert st.read() == 1 and not torch.isfinite(k[0, 1, 1, 63])


def attend(L, s, heads, group, dim, dtype, seed=0, scale=None, strided=False):
    """q, caches filled with N(0, 1), the planned step run through attention; (out, q, k, v, cache)."""
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = getattr(torch, dtype)
    k, v = (torch.randn((s.pages, heads, s.page, dim), device="cuda", generator=gen).to(kind) for _ in range(2))
    q = torch.randn((s.tokens, heads * group + (2 if strided else 0), dim), device="cuda", generator=gen).to(kind)[:, :heads * group]
    s.plan()
    cache = L.kv_cache_of(k, v)
    out = torch.full((s.tokens, heads * group, dim), 7.0, dtype=kind, device="cuda")
    L.attention_paged(cache, s.step, q, scale or dim ** -0.5, s.status, out=out)
    return out, q, k, v, cache


def check_attention(s, out, q, k, v, scale=None):
    import torch
    dim = q.shape[-1]
    want, spread, score = O.attention(q, k, v, s.table, s.cached, s.want["offsets"], s.masks(), scale or dim ** -0.5)
    rows = s.want["offsets"][-1]
    keys = max(c + f for c, f in zip(s.cached, s.fresh))
    off = (out.double() - want)[:rows].abs()
    room = O.attention_bound(out.dtype, want, spread, score, keys, dim)[:rows]
    assert bool((off <= room).all()), (float((off / room).max()), float(off.max()))
    assert bool((out[rows:] == 7.0).all())                       # padding rows are left as they were
    assert torch.isfinite(out[:rows]).all()


DECODE = [([0], [1]), ([1], [1]), ([15, 16, 17], [1, 1, 1]), ([63, 64, 127, 128, 129], [1] * 5), ([700, 0, 3], [1, 0, 1]), ([5000, 40, 1999], [1, 1, 1])]
CHAINS = [([0], [2]), ([126], [4]), ([0, 250, 31], [3, 4, 1]), ([1000, 5], [2, 3])]
MANY = [([0], [17]), ([0], [129]), ([100], [64]), ([127, 0, 600], [33, 40, 1]), ([300, 1], [300, 70]), ([2000], [40])]
TREES = [([0], [1]), ([0], [64]), ([129], [33]), ([500, 0, 64], [64, 5, 31]), ([3000, 1], [16, 64])]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("heads,group,dim,page", [(1, 1, 64, 16), (2, 4, 128, 16), (3, 8, 128, 64), (2, 5, 64, 48), (1, 16, 256, 32), (4, 2, 256, 256), (1, 7, 128, 4096)])
@pytest.mark.parametrize("which", range(len(DECODE)))
def test_attention_one_token(L, which, heads, group, dim, page, dtype):
    cached, fresh = DECODE[which]
    s = Step(L, cached, fresh, page, seed=which, extra_tokens=2)
    out, q, k, v, _ = attend(L, s, heads, group, dim, dtype, which, strided=which % 2 == 1)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v)


@pytest.mark.parametrize("heads,group,dim,page,dtype", [(2, 4, 128, 16, "bfloat16"), (1, 5, 64, 48, "float16"), (2, 3, 256, 64, "bfloat16"), (1, 24, 128, 32, "float16")])
@pytest.mark.parametrize("which", range(len(CHAINS)))
def test_attention_chain(L, which, heads, group, dim, page, dtype):
    cached, fresh = CHAINS[which]
    s = Step(L, cached, fresh, page, seed=which, extra_tokens=1)
    out, q, k, v, _ = attend(L, s, heads, group, dim, dtype, which)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v)


@pytest.mark.parametrize("heads,group,dim,page,dtype", [(2, 4, 128, 64, "bfloat16"), (1, 7, 64, 16, "float16"), (2, 2, 256, 128, "bfloat16"), (1, 16, 128, 48, "float16"),
                                                        (3, 1, 64, 256, "bfloat16")])
@pytest.mark.parametrize("which", range(len(MANY)))
def test_attention_prompt(L, which, heads, group, dim, page, dtype):
    cached, fresh = MANY[which]
    s = Step(L, cached, fresh, page, seed=which, extra_tokens=9)
    out, q, k, v, _ = attend(L, s, heads, group, dim, dtype, which, strided=which % 2 == 0)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v)


@pytest.mark.parametrize("heads,group,dim,page,dtype", [(2, 4, 128, 64, "bfloat16"), (1, 1, 64, 16, "float16"), (1, 2, 256, 48, "bfloat16"), (2, 8, 128, 16, "float16")])
@pytest.mark.parametrize("shape", ["random", "chain", "star"])
@pytest.mark.parametrize("which", range(len(TREES)))
def test_attention_tree(L, which, shape, heads, group, dim, page, dtype):
    cached, fresh = TREES[which]
    s = Step(L, cached, fresh, page, seed=which, tree=shape, extra_tokens=4)
    out, q, k, v, _ = attend(L, s, heads, group, dim, dtype, which)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v)


@pytest.mark.parametrize("dtype,dim,group", [("bfloat16", 128, 4), ("float16", 64, 5), ("bfloat16", 256, 3), ("float16", 128, 7), ("bfloat16", 64, 2)])
@pytest.mark.parametrize("tree", [None, "random"])
@pytest.mark.parametrize("most", [1, 3, 64])
def test_attention_many_requests(L, most, tree, dtype, dim, group):
    """Shares of one CTA that hold ends, whole items and beginnings, of one tile of rows and of two, of requests with and without
    fresh tokens; twice, with the same bits."""
    import torch
    rng = np.random.default_rng(most)
    requests = 45
    fresh = (rng.integers(1, most + 1, requests) * (rng.random(requests) < 0.9)).tolist()
    fresh[0] = most
    cached = (2500 * rng.random(requests) ** 3).astype(int).tolist()
    s = Step(L, cached, fresh, 32, seed=most, tree=tree)
    out, q, k, v, cache = attend(L, s, 4, group, dim, dtype, most)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v)
    again = L.attention_paged(cache, s.step, q, dim ** -0.5, s.status)
    assert torch.equal(again[:sum(fresh)], out[:sum(fresh)])


@pytest.mark.parametrize("scale", [1e-3, 3.0])
@pytest.mark.parametrize("fresh", [1, 40])
def test_attention_scales(L, scale, fresh):
    """Scores from nearly equal ones to ones of which a single key takes all the weight."""
    s = Step(L, [777], [fresh], 32)
    out, q, k, v, _ = attend(L, s, 2, 4, 128, "bfloat16", scale=scale)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v, scale)


@pytest.mark.parametrize("fresh,group", [(1, 4), (33, 4), (40, 8)])
def test_attention_growing_scores(L, fresh, group):
    """Keys whose scores grow along the cache: the running maximum moves in every block, far beyond one exponent."""
    import torch
    s = Step(L, [1500], [fresh], 16)
    _, q, k, v, cache = attend(L, s, 1, group, 128, "bfloat16")
    for j in range(1500 + fresh):
        k[s.table[0, j // 16], 0, j % 16] = (0.02 * j) * torch.sign(q[0, 0])
    q.copy_(q[0, 0].abs() * torch.sign(q[0, 0]))
    out = torch.full_like(q, 7.0)
    L.attention_paged(cache, s.step, q, 0.02, s.status, out=out)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v, 0.02)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tree", [None, "star"])
@pytest.mark.parametrize("cached,fresh,group", [(20, 3, 2), (20, 30, 4), (130, 64, 8), (0, 64, 1)])
def test_attention_unseen_keys_have_no_influence(L, cached, fresh, group, tree, dim):
    """NaN, infinities and the largest numbers behind a request's end, in other requests' pages, and in the fresh tokens that a row
    does not see; the row of a token whose own value is NaN is reported and NaN."""
    import torch
    s = Step(L, [cached], [fresh], 16, tree=tree)
    _, q, k, v, cache = attend(L, s, 2, group, dim, "bfloat16")
    for at, x in ((k, float("nan")), (v, float("inf"))):
        clean = at.clone()
        at.fill_(x)
        for j in range(cached + fresh):
            at[s.table[0, j // 16], :, j % 16] = clean[s.table[0, j // 16], :, j % 16]
    out = torch.full_like(q, 7.0)
    L.attention_paged(cache, s.step, q, dim ** -0.5, s.status, out=out)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v)
    # the last token's value: only the rows that see it
    last = cached + fresh - 1
    for x in (float("nan"), float("inf"), 3e38):
        v2 = v.clone()
        v2[s.table[0, last // 16], :, last % 16] = x
        got = torch.full_like(q, 7.0)
        s.status.reset()
        L.attention_paged(L.kv_cache_of(k, v2), s.step, q, dim ** -0.5, s.status, out=got)
        assert torch.equal(got[:fresh - 1], out[:fresh - 1])
        if x != 3e38:
            assert s.status.read() == 1 and not torch.isfinite(got[fresh - 1]).any()
    # the last token's key
    k2 = k.clone()
    k2[s.table[0, last // 16], :, last % 16] = float("nan")
    got = torch.full_like(q, 7.0)
    s.status.reset()
    L.attention_paged(L.kv_cache_of(k2, v), s.step, q, dim ** -0.5, s.status, out=got)
    assert s.status.read() == 1 and torch.equal(got[:fresh - 1], out[:fresh - 1]) and not torch.isfinite(got[fresh - 1]).any()


@pytest.mark.parametrize("fresh,group", [(4, 2), (30, 4), (64, 8)])
def test_attention_rows_that_see_nothing(L, fresh, group):
    """Masks of zero over an empty cache: zeros, no status; over a cache they see just that."""
    import torch
    for cached in (0, 40):
        s = Step(L, [cached, 5], [fresh, 3], 16, tree="random")
        out, q, k, v, cache = attend(L, s, 2, group, 64, "bfloat16")
        for t in range(0, fresh, 3):
            s.step.ancestors_tensor[t] = 0
            s.want["ancestors"][t] = 0
        out.fill_(7.0)
        L.attention_paged(cache, s.step, q, 0.125, s.status, out=out)
        assert s.status.read() == 0
        check_attention(s, out, q, k, v)
        if cached == 0:
            assert bool((out[0] == 0).all())
    assert torch.isfinite(out).all()


def test_attention_bad_pages_and_lengths(L):
    """A page outside the cache counts as unseen and is reported; lengths above their bounds and offsets of no plan are reported
    and read nothing outside."""
    import torch
    for fresh in (1, 40):
        for bad in (-1, 1 << 30, 10 ** 6):
            s = Step(L, [100], [fresh], 16)
            _, q, k, v, cache = attend(L, s, 2, 4, 64, "bfloat16")
            s.table_dev[0, 2] = bad
            out = torch.full_like(q, 7.0)
            L.attention_paged(cache, s.step, q, 0.125, s.status, out=out)
            assert s.status.read() == 2
            at = [j for j in range(100 + fresh) if j // 16 != 2]
            kk, vv = (torch.stack([x[s.table[0, j // 16], :, j % 16] for j in at], 1)[None] for x in (k, v))      # one page of what is left
            pad = 64 * 3 - len(at)
            kk, vv = (torch.nn.functional.pad(x[0], (0, 0, 0, pad)).unsqueeze(0) for x in (kk, vv))
            want, spread, score = O.attention(q, kk, vv, [[0]], [100 - 16], [0, fresh], None, 0.125)
            assert bool(((out.double() - want).abs() <= O.attention_bound(out.dtype, want, spread, score, 140, 64)).all())
        for change in ("cached", "offsets", "negative", "far"):
            s = Step(L, [100, 50], [fresh, fresh], 16)
            _, q, k, v, cache = attend(L, s, 2, 4, 64, "bfloat16")
            if change == "cached":
                s.cached_dev[0] = 10 ** 9
            elif change == "negative":
                s.cached_dev[1] = -5
            elif change == "offsets":
                s.step.offsets_tensor[1] = -3
            else:
                s.step.offsets_tensor[2] = 1 << 30
            L.attention_paged(cache, s.step, q, 0.125, s.status)
            assert s.status.read() == 2


@pytest.mark.parametrize("fresh", [1, 40])
def test_attention_pages_past_32_bits(L, fresh):
    """A cache of more than 2^32 bytes a side, the request's pages at both ends of it."""
    import torch
    heads, dim, page = 2, 128, 64
    pages = (5 << 30) // (heads * page * dim * 2)
    s = Step(L, [300], [fresh], page)
    n = up(300 + fresh, page)
    ids = [0, pages - 1, pages // 2, pages - 2, 1, pages - 5][:n]
    s.pages = pages
    s.table[0, :n] = ids
    s.table_dev.copy_(ints(s.table))
    s.free_dev = ints([ids[i] for i in range(up(300, page), n)] or [2])
    k, v = (torch.empty((pages, heads, page, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    s.plan()
    cache, slots = L.kv_cache_of(k, v), []
    for j in range(300 + fresh):
        slots.append(ids[j // page] * page + j % page)
    rows = torch.randn((300 + fresh, 2, heads, dim), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    L.kv_append(cache, ints(slots, torch.int64), rows[:, 0], rows[:, 1], s.status)
    assert s.step.slots_tensor.tolist() == slots[300:]
    q = torch.randn((fresh, heads * 4, dim), device="cuda").to(torch.bfloat16)
    out = L.attention_paged(cache, s.step, q, dim ** -0.5, s.status)
    assert s.status.read() == 0
    at = ints(ids).long()
    s.table = np.arange(n, dtype=np.int32)[None]
    check_attention(s, out, q, k[at], v[at])


@pytest.mark.parametrize("group", [32, 128, 130, 256])
@pytest.mark.parametrize("fresh", [1, 3])
def test_attention_large_groups(L, fresh, group):
    """Groups of which a tile holds several tokens, one, a token and a part, and half a token."""
    s = Step(L, [200, 7], [fresh, 1], 16, extra_tokens=1)
    out, q, k, v, _ = attend(L, s, 1, group, 64, "bfloat16")
    assert s.status.read() == 0
    check_attention(s, out, q, k, v)


@pytest.mark.parametrize("fresh", [1, 20])
def test_attention_of_shared_pages(L, fresh):
    """Requests whose tables begin with the same pages: a common prefix, stored once."""
    import torch
    s = Step(L, [160, 160, 96], [fresh, fresh, fresh], 32, extra_pages=9)
    for r in (1, 2):
        s.table[r, :3] = s.table[0, :3]
    s.table_dev.copy_(ints(s.table))
    out, q, k, v, _ = attend(L, s, 2, 4, 128, "float16")
    assert s.status.read() == 0
    check_attention(s, out, q, k, v)


@pytest.mark.parametrize("fresh,tree", [(5, None), (40, "random")])
def test_attention_behind_other_kernels(L, fresh, tree):
    """Plan, append and attention of many steps in flight on one stream, each writing what the next one reads, with nothing waited for
    between them: the last step's results are those of the same steps one at a time."""
    import torch
    def go(wait):
        s = Step(L, [0, 0], [fresh, fresh], 16, tree=tree, extra_pages=90, extra_width=30)
        gen = torch.Generator(device="cuda")
        gen.manual_seed(5)
        k, v = (torch.zeros((s.pages, 2, 16, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        cache, geometry, outs = L.kv_cache_of(k, v), L.kv_geometry_of(s.pages, 16), []
        s.step.longest = 16 * s.width
        ws, used, rows = L.attention_paged_workspace(cache, s.step, 8), torch.empty(1, dtype=torch.int32, device="cuda"), torch.empty((s.tokens, 2, 2, 64), device="cuda")
        q = torch.empty((s.tokens, 8, 64), dtype=torch.bfloat16, device="cuda")
        free = s.free_dev
        for i in range(8):
            rows.normal_(generator=gen)
            q.normal_(generator=gen)
            L.kv_plan(geometry, s.step, free, s.status, used)
            L.kv_append(cache, s.step.slots_tensor, rows[:, 0], rows[:, 1], s.status)
            outs.append(L.attention_paged(cache, s.step, q, 0.125, s.status, workspace=ws))
            before, after = up(fresh * i, 16), up(fresh * (i + 1), 16)
            free = free[2 * (after - before):].contiguous()
            s.cached_dev += fresh
            if wait:
                torch.cuda.synchronize()
        assert s.status.read() == 0
        return outs
    for a, b in zip(go(False), go(True)):
        assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("position", [0, 777, 1499])
def test_attention_of_a_contiguous_cache(L, position):
    """One page per session is the cache that attention_gqa_decode reads: the same values, once rounded."""
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(position)
    sessions, heads, dim, context = 3, 2, 128, 1504
    k, v = (torch.randn((sessions, heads, context, dim), device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
    q = torch.randn((sessions, 4 * heads, dim), device="cuda", generator=gen).to(torch.bfloat16)
    st = L.Status()
    want = L.attention_gqa_decode(q, k, v, position, dim ** -0.5, st)
    step = L.kv_step_of(ints([position] * sessions), ints([1] * sessions), ints([[i] for i in range(sessions)]), sessions, 1, context)
    L.kv_plan(L.kv_geometry_of(sessions, context), step, ints([0, 1, 2]), st)
    out = L.attention_paged(L.kv_cache_of(k, v), step, q, dim ** -0.5, st)
    assert st.read() == 0
    u = torch.finfo(torch.bfloat16).eps / 2
    mean = L.attention_gqa_decode(q, k, v.abs(), position, dim ** -0.5, st).double()
    assert bool(((out.double() - want.double()).abs() <= 1.01 * u * (want.double().abs() + mean) + 1e-6).all())


@pytest.mark.parametrize("fresh", [1, 24])
def test_attention_captured_and_replayed_with_other_lengths(L, fresh):
    """A step captured once and replayed while the lengths, the pages and the rows change; two such graphs beside one another."""
    import torch
    page, heads, group, dim, longest = 16, 2, 4, 128, 600
    graphs = []
    for g in range(2):
        s = Step(L, [longest - fresh, 3], [fresh, fresh], page, seed=g, extra_pages=40)
        out, q, k, v, cache = attend(L, s, heads, group, dim, "bfloat16", g)
        ws, used = L.attention_paged_workspace(cache, s.step, heads * group), torch.empty(1, dtype=torch.int32, device="cuda")
        rows = torch.randn((s.tokens, 2, heads, dim), device="cuda")
        geometry = L.kv_geometry_of(s.pages, page)

        def run():
            L.kv_plan(geometry, s.step, s.free_dev, s.status, used)
            L.kv_append(cache, s.step.slots_tensor, rows[:, 0], rows[:, 1], s.status)
            L.attention_paged(cache, s.step, q, dim ** -0.5, s.status, workspace=ws, out=out)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            run()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                run()
        graphs.append((s, out, q, k, v, rows, graph, stream))
    torch.cuda.synchronize()
    for cached, lens in (([500, 17], [fresh, 1]), ([0, 0], [1, fresh]), ([33, 550 - fresh], [0, fresh])):
        for s, out, q, k, v, rows, graph, stream in graphs:
            with torch.cuda.stream(stream):
                order = s.rng.permutation(s.pages).astype(np.int32)
                s.cached, s.fresh, at = cached, lens, 0
                for r in range(2):
                    h = up(cached[r], page)
                    s.table[r, :h] = order[at:at + h]
                    at += h
                s.free = order[at:at + s.free_dev.numel()]
                assert len(s.free) == s.free_dev.numel()
                for dev, x in ((s.cached_dev, cached), (s.fresh_dev, lens), (s.table_dev, s.table), (s.free_dev, s.free)):
                    dev.copy_(ints(x))
                rows.normal_()
                out.fill_(7.0)
                graph.replay()
        torch.cuda.synchronize()
        for s, out, q, k, v, rows, graph, stream in graphs:
            s.want = O.plan(cached, lens, s.table, s.free, page, s.tokens)
            assert s.status.read() == 0 and s.step.slots_tensor.tolist() == s.want["slots"]
            for t, slot in enumerate(s.want["slots"]):
                if slot >= 0:
                    assert torch.equal(k[slot // page, :, slot % page], rows[t, 0].to(k.dtype))
            check_attention(s, out, q, k, v)


def test_calls_on_two_streams(L):
    """Two sessions' steps in flight at once, each on a stream of its own, many times over."""
    import torch
    made = []
    for g in range(2):
        s = Step(L, [900, 100 * g], [1 + 30 * g, 2], 32, seed=g)
        out, q, k, v, cache = attend(L, s, 4, 4, 128, "bfloat16", g)
        made.append((s, out, q, k, v, cache, L.attention_paged_workspace(cache, s.step, 16), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for s, out, q, k, v, cache, ws, stream in made:
            with torch.cuda.stream(stream):
                out.fill_(7.0)
                L.attention_paged(cache, s.step, q, 128 ** -0.5, s.status, workspace=ws, out=out)
    torch.cuda.synchronize()
    for s, out, q, k, v, *_ in made:
        assert s.status.read() == 0
        check_attention(s, out, q, k, v)


# ---- logits -----------------------------------------------------------------------------------------------------------

def edit_case(L, vocabulary, fresh, tree, dtype, history=200, biases=7, grammar=True, seed=0, stride=0, padding=0):
    import torch
    rng = np.random.default_rng(seed)
    R, rows = len(fresh), sum(fresh) + padding
    pick = lambda n: np.minimum((vocabulary ** rng.random(n)).astype(np.int64) - 1, vocabulary - 1)  # noqa: E731
    hist = [pick(int(rng.integers(0, history + 1))).tolist() for _ in range(R)]
    for h in hist[1:]:
        h.insert(len(h) // 2, -1)                                # padding among the words
    prompt = [int(rng.integers(0, len(h) + 1)) for h in hist]
    rep, pres, freq = rng.uniform(0.8, 1.4, R).astype(np.float32), rng.uniform(-0.5, 1, R).astype(np.float32), rng.uniform(0, 0.5, R).astype(np.float32)
    bias = [[(int(w), float(np.float32(x))) for w, x in zip(pick(biases), rng.normal(0, 5, biases))] for _ in range(R)]      # words twice: the last counts
    off = np.concatenate([[0], np.cumsum(fresh)]).tolist()
    request = sum(([r] * f for r, f in enumerate(fresh)), []) + [-1] * padding
    drafted = pick(rows).tolist()
    parents = O.parents_of(rng, fresh, "random")
    masks = O.plan([0] * R, fresh, np.zeros((R, 1 + max(fresh) // 16), np.int32), list(range(rows + R)), 16, rows, parents if tree else None)["ancestors"]
    paths = [[] if r < 0 else [drafted[off[r] + j] for j in range(fresh[r]) if (masks[t] >> j & 1 if tree else j <= t - off[r])] for t, r in enumerate(request)]
    words = up(vocabulary, 32)
    mask = rng.integers(-2 ** 31, 2 ** 31, (rows, words + 1)).astype(np.int32) if grammar else None
    if grammar:
        mask[0] = 0                                              # nothing allowed
    kind = getattr(torch, dtype)
    values = torch.tensor(rng.normal(0, 3, (rows, vocabulary + stride)).astype(np.float32), device="cuda").to(kind)
    policy = L.logits_policy_of(vocabulary, ints(sum(hist, []) or [0]), ints(np.concatenate([[0], np.cumsum([len(h) for h in hist])]).tolist()), ints(prompt),
                                ints(rep, torch.float32), ints(pres, torch.float32), ints(freq, torch.float32),
                                ints([w for b in bias for w, _ in b] or [0]), ints([x for b in bias for _, x in b] or [0.0], torch.float32),
                                ints([biases * r for r in range(R + 1)]))
    drafts = L.logits_drafts_of(ints(drafted), ints(request), ints(off), ints([O.signed(m) for m in masks], torch.int64) if tree else None, tree=tree)
    want = O.logits(values[:, :vocabulary].double().cpu().numpy(), request, hist, prompt, rep.astype(np.float64), pres.astype(np.float64), freq.astype(np.float64),
                    bias, paths, mask, vocabulary)
    return policy, drafts, values[:, :vocabulary], None if mask is None else ints(mask), want, request


def check_edit(out, want, request, before):
    import torch
    got, live = out.double().cpu().numpy(), np.array([r >= 0 for r in request])
    assert np.array_equal(np.isneginf(got[live]), np.isneginf(want[live]))
    u, f = torch.finfo(out.dtype).eps / 2, torch.finfo(torch.float32).eps / 2
    fine = np.isfinite(want) & live[:, None]
    # half a step of the result, and half an f32 step for each of the five operations on values of at most 3 sigma and the penalties' sizes
    scale = np.maximum(np.abs(want[fine]), 200.0)
    assert (np.abs(got[fine] - want[fine]) <= 1.01 * u * np.abs(want[fine]) + 5 * f * scale).all()
    assert np.array_equal(got[~live], before.double().cpu().numpy()[~live])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("vocabulary,fresh,stride,grammar", [(1, [1], 0, True), (31, [1, 2], 0, True), (1000, [1], 3, True), (4099, [3, 1, 0, 5], 1, True),
                                                             (32001, [2, 7], 0, False), (129280, [1], 0, True), (9000, [64, 20, 1], 8, True), (5000, [1] * 40, 5, True)])
def test_logits(L, vocabulary, fresh, stride, grammar, tree, dtype):
    import torch
    policy, drafts, x, mask, want, request = edit_case(L, vocabulary, fresh, tree, dtype, grammar=grammar, seed=vocabulary, stride=stride, padding=2)
    st = L.Status()
    out = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda")
    before = out.clone()
    L.logits_edit(policy, drafts, x, st, grammar=mask, out=out)
    assert st.read() == 0
    check_edit(out, want, request, before)
    same = x.clone() if stride else x
    before = same.clone()
    L.logits_edit(policy, drafts, same, st, grammar=mask, out=same)              # in place
    assert st.read() == 0
    live = [t for t, r in enumerate(request) if r >= 0]
    assert torch.equal(same[live], out[live]) and torch.equal(same[-2:], before[-2:])


def test_logits_long_history_and_no_history(L):
    import torch
    policy, drafts, x, mask, want, request = edit_case(L, 50000, [5, 1], True, "float32", history=30000, seed=3)
    st = L.Status()
    out = torch.empty_like(x)
    L.logits_edit(policy, drafts, x, st, grammar=mask, out=out)
    assert st.read() == 0
    check_edit(out, want, request, out)
    # only a grammar; nothing at all: a copy
    rows = x.shape[0]
    bare = L.logits_policy_of(50000, requests=rows)
    plain = L.logits_drafts_of(rows=rows)
    out = L.logits_edit(bare, plain, x, st, grammar=mask)
    bits = (mask[:, torch.arange(50000, device="cuda") // 32] >> (torch.arange(50000, device="cuda") % 32)) & 1
    assert st.read() == 0 and torch.equal(out, torch.where(bits == 1, x, torch.full_like(x, -float("inf"))))
    assert torch.equal(L.logits_edit(bare, plain, x, st), x) and st.read() == 0


@pytest.mark.parametrize("vocabulary,biases", [(700, 500), (40000, 3000)])
def test_logits_many_biases(L, vocabulary, biases):
    """More entries than a CTA lists, words among them several times: the last entry counts."""
    import torch
    policy, drafts, x, mask, want, request = edit_case(L, vocabulary, [2, 1], False, "float32", biases=biases, seed=biases)
    st = L.Status()
    out = L.logits_edit(policy, drafts, x, st, grammar=mask)
    assert st.read() == 0
    check_edit(out, want, request, out)


def test_logits_more_words_than_a_table_holds(L):
    """A history with tens of thousands of different words, over one row and over several, with paths and biases among them."""
    import torch
    for fresh, tree in (([1], False), ([5, 3], False), ([20], True)):
        policy, drafts, x, mask, want, request = edit_case(L, 60000, fresh, tree, "float32", history=10, biases=2000, seed=len(fresh))
        words = torch.randperm(60000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(torch.int32)
        R = len(fresh)
        p2 = L.logits_policy_of(60000, words, ints([0] + [60000] * R), ints([40000] * R), *policy._keep[3:])
        st = L.Status()
        out = L.logits_edit(p2, drafts, x, st, grammar=mask)
        assert st.read() == 0
        k = policy._keep
        hist = [words.tolist()] + [[]] * (R - 1)
        off, bo = drafts._keep[2].tolist(), k[8].tolist()
        bias = [list(zip(k[6].tolist()[bo[r]:bo[r + 1]], k[7].tolist()[bo[r]:bo[r + 1]])) for r in range(R)]
        drafted, masks = drafts._keep[0].tolist(), drafts._keep[3].tolist() if tree else None
        paths = [[] if r < 0 else [drafted[off[r] + j] for j in range(fresh[r]) if (masks[t] >> j & 1 if tree else j <= t - off[r])] for t, r in enumerate(request)]
        f64 = [k[i].double().cpu().numpy() for i in (3, 4, 5)]
        want = O.logits(x.double().cpu().numpy(), request, hist, [40000] * R, *f64, bias, paths, mask.cpu().numpy(), 60000)
        check_edit(out, want, request, out)


def test_logits_infinities_and_nan(L):
    """Infinities pass; NaN in a place that the grammar forbids is gone, in an allowed one it stays and is reported."""
    import torch
    x = torch.randn((2, 5000), device="cuda")
    x[0, 7], x[0, 8], x[1, 9] = -float("inf"), float("inf"), float("nan")
    mask = torch.full((2, 157), -1, dtype=torch.int32, device="cuda")
    mask[1, 0] = ~(1 << 9)
    policy, drafts, st = L.logits_policy_of(5000, ints([7, 8, 9, 9]), ints([0, 3, 4]), repetition=ints([1.5, 1.5], torch.float32)), L.logits_drafts_of(rows=2), L.Status()
    out = L.logits_edit(policy, drafts, x, st, grammar=mask)
    assert st.read() == 0 and out[0, 7] == -float("inf") and out[0, 8] == float("inf") and out[1, 9] == -float("inf")
    out = L.logits_edit(policy, drafts, x, st)
    assert st.read() == 1 and torch.isnan(out[1, 9])


def test_logits_reports_bad_words_requests_and_penalties(L):
    import torch
    x = torch.randn((2, 5000), device="cuda")
    def run(policy=None, drafts=None):
        st = L.Status()
        out = L.logits_edit(policy or L.logits_policy_of(5000, requests=2), drafts or L.logits_drafts_of(rows=2), x, st)
        return st.read(), out
    assert run()[0] == 0
    assert run(L.logits_policy_of(5000, ints([1, 5000]), ints([0, 1, 2])))[0] == 2
    assert run(L.logits_policy_of(5000, ints([1, 2]), ints([0, 2, 1])))[0] == 2
    for r in (0.0, -1.0, float("nan"), float("inf")):
        code, out = run(L.logits_policy_of(5000, ints([1, 2]), ints([0, 1, 2]), repetition=ints([r, 1.0], torch.float32)))
        assert code == 2
    assert run(L.logits_policy_of(5000, bias_tokens=ints([5001]), bias_values=ints([1.0], torch.float32), bias_offsets=ints([0, 0, 1])))[0] == 2
    code, out = run(drafts=L.logits_drafts_of(row_request=ints([1, 2])))
    assert code == 2
    assert run(drafts=L.logits_drafts_of(ints([1, 5000]), ints([0, 1]), ints([0, 1, 2])))[0] == 2
    assert run(drafts=L.logits_drafts_of(ints([1, 2]), ints([0, 1]), ints([0, 2, 1])))[0] == 2


# ---- the four in a row ------------------------------------------------------------------------------------------------

def test_steps_in_a_row(L):
    """A prompt, decode steps, and drafted trees of which a path is kept, for three requests over one cache: what the pages hold and
    what attention and the edits give after each step, against restatements that keep every request's history as a plain list."""
    import torch
    torch.manual_seed(0)
    rng = np.random.default_rng(0)
    R, page, H, G, D, V, width, pages = 3, 16, 2, 4, 64, 1000, 12, 40
    k, v = (torch.full((pages, H, page, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache, st = L.kv_cache_of(k, v), L.Status()
    table = torch.full((R, width), -1, dtype=torch.int32, device="cuda")
    free = list(rng.permutation(pages))
    cached, kv, text = [0] * R, [[] for _ in range(R)], [[] for _ in range(R)]
    for kind, fresh in (("prompt", [37, 20, 70]), ("decode", [1, 1, 1]), ("tree", [9, 16, 4]), ("decode", [1, 0, 1]), ("tree", [5, 5, 5]), ("chain", [3, 2, 4])):
        n = sum(fresh)
        tree = kind == "tree"
        parents = O.parents_of(rng, fresh, "random") if tree else None
        step = L.kv_step_of(ints(cached), ints(fresh), table, n + 2, max(fresh), max(c + f for c, f in zip(cached, fresh)), parents=ints(parents + [-1, -1]) if tree else None)
        used = int(L.kv_plan(L.kv_geometry_of(pages, page), step, ints(free), st)[0])
        free = free[used:]
        rows, q = torch.randn((n + 2, 2, H, D), device="cuda"), torch.randn((n + 2, H * G, D), device="cuda").to(torch.bfloat16)
        L.kv_append(cache, step.slots_tensor, rows[:, 0], rows[:, 1], st)
        out = L.attention_paged(cache, step, q, D ** -0.5, st)
        drafted = rng.integers(0, V, n + 2).tolist()
        flat = sum(text, [])
        policy = L.logits_policy_of(V, ints(flat or [0]), ints(np.concatenate([[0], np.cumsum([len(x) for x in text])]).tolist()), frequency=ints([0.25] * R, torch.float32))
        x = torch.randn((n + 2, V), device="cuda")
        edited = L.logits_edit(policy, L.logits_drafts_of(ints(drafted), step.row_request_tensor, step.offsets_tensor, step.ancestors_tensor, tree=tree), x, st)
        assert st.read() == 0
        off, masks = step.offsets_tensor.tolist(), [m % (1 << 64) for m in step.ancestors_tensor.tolist()] if tree else None
        # restatement: each row's keys and values as one list
        for r in range(R):
            for t in range(off[r], off[r + 1]):
                on = [j for j in range(fresh[r]) if (masks[t] >> j & 1 if tree else j <= t - off[r])]
                both = torch.stack(kv[r] + [rows[off[r] + j].to(torch.bfloat16) for j in on])
                want, spread, score = O.attention(q[t:t + 1], both[:, 0].transpose(0, 1)[None], both[:, 1].transpose(0, 1)[None], [[0]], [len(both) - 1], [0, 1], None, D ** -0.5)
                assert bool(((out[t:t + 1].double() - want).abs() <= O.attention_bound(out.dtype, want, spread, score, len(both), D)).all())
                count = np.bincount(text[r] + [drafted[off[r] + j] for j in on], minlength=V)
                assert np.allclose(edited[t].cpu().numpy(), x[t].cpu().numpy() - 0.25 * count, rtol=0, atol=2e-6)
        # what is kept: everything, or the path to a node of the tree, stored again behind the cached tokens
        slots, source = [], []
        for r in range(R):
            keep = [j for j in range(fresh[r]) if not tree or masks[off[r + 1] - 1] >> j & 1]
            for i, j in enumerate(keep):
                at = cached[r] + i
                slots.append(int(table[r, at // page]) * page + at % page)
                source.append(off[r] + j)
                kv[r].append(rows[off[r] + j].to(torch.bfloat16))
                text[r].append(drafted[off[r] + j])
            if tree:                                             # pages past the kept tokens are free again
                for c in range(up(cached[r] + len(keep), page), up(cached[r] + fresh[r], page)):
                    free.append(int(table[r, c]))
            cached[r] += len(keep)
        if tree:
            kept = rows[ints(source).long()]
            L.kv_append(cache, ints(slots, torch.int64), kept[:, 0], kept[:, 1], st)
        assert st.read() == 0
