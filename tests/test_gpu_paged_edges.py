"""A serving step over a paged cache on a B200, at its edges: word lists that do not fit a table, requests whose lengths are bad, weights far
below the largest, against plain restatements in 64 bits."""
import numpy as np
import pytest

import paged_oracle as O
from test_gpu_paged import L, Step, attend, check_attention, check_edit, ints, up  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- logits: more words than a table holds ----------------------------------------------------------------------------

TABLE = 12288                                                    # words that the largest table takes


def word_lists():
    rng = np.random.default_rng(5)
    return {
        "even": np.arange(13000) * 2, "consecutive": np.arange(2 * TABLE + 1), "random": rng.permutation(60000)[:2 * TABLE],
        "even_and_a_few_odd": np.concatenate([np.arange(25000) * 2, np.arange(100) * 2 + 1]), "uneven": np.concatenate([np.arange(14000) * 2, np.arange(3000) * 2 + 1]),
        "fours": np.arange(15000) * 4, "four_tables": rng.permutation(60000)[:4 * TABLE], "one_table": np.arange(TABLE), "one_more": np.arange(TABLE + 1) * 3,
    }


@pytest.mark.parametrize("where", ["history", "biases"])
@pytest.mark.parametrize("name", sorted(word_lists()))
@pytest.mark.parametrize("rows", [1, 50, 80, 170])
def test_logits_words_that_do_not_fit_a_table(L, rows, name, where):  # noqa: F811
    """Every word is edited once, however unevenly the words fall on the parts that are counted one after the other; rows enough that the launch
    begins with many parts, two, one, and one for two rows; out of place and in place."""
    import torch
    V, words = 60000, word_lists()[name]
    rng = np.random.default_rng(rows)
    words = rng.permutation(words).astype(np.int32)
    values = rng.normal(0, 5, len(words)).astype(np.float32)
    x = torch.randn((rows, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(rows))
    want = x.double().cpu().numpy()
    if where == "history":
        policy = L.logits_policy_of(V, ints(words), ints([0, len(words)]), ints([len(words) // 3]), *(ints([p], torch.float32) for p in (1.25, 0.5, 0.125)))
        made = np.zeros(V)
        made[words[len(words) // 3:]] = 1
        at = want[:, words]
        want[:, words] = np.where(at > 0, at / 1.25, at * 1.25)
        want -= 0.625 * made
    else:
        policy = L.logits_policy_of(V, bias_tokens=ints(words), bias_values=ints(values, torch.float32), bias_offsets=ints([0, len(words)]))
        want[:, words] += values
    drafts, st = L.logits_drafts_of(row_request=ints([0] * rows)), L.Status()
    out = L.logits_edit(policy, drafts, x, st)
    assert st.read() == 0
    check_edit(out, want, [0] * rows, out)
    L.logits_edit(policy, drafts, x, st, out=x)
    assert st.read() == 0 and torch.equal(x, out)


@pytest.mark.parametrize("rows", [1, 80])
def test_logits_long_bias_lists(L, rows):  # noqa: F811
    """Lists of tens of thousands of entries, every word several times: the last entry counts, and the work grows with the entries, not with
    their product with the words (40 000 entries of 10 000 words in 80 rows took 28 ms that way)."""
    import torch
    V, n, words = 50000, 40000, 10000
    rng = np.random.default_rng(rows)
    tokens, values = rng.integers(0, words, n).astype(np.int32) * 5, rng.normal(0, 5, n).astype(np.float32)
    tokens[:words] = rng.permutation(words) * 5                  # (some words only at the list's beginning)
    x = torch.randn((rows, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(rows))
    want, last = x.double().cpu().numpy(), dict(zip(tokens.tolist(), values.tolist()))
    want[:, list(last)] += np.array(list(last.values()))
    policy = L.logits_policy_of(V, bias_tokens=ints(tokens), bias_values=ints(values, torch.float32), bias_offsets=ints([0, n]))
    drafts, st = L.logits_drafts_of(row_request=ints([0] * rows)), L.Status()
    out = L.logits_edit(policy, drafts, x, st)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    L.logits_edit(policy, drafts, x, st, out=out)
    end.record()
    assert st.read() == 0
    check_edit(out, want, [0] * rows, out)
    assert begin.elapsed_time(end) < (10.0 if rows == 80 else 2.0), begin.elapsed_time(end)


@pytest.mark.parametrize("lists", [[2561, 0, 0], [7000, 3, 500], [8192, 9000], [2560, 2560], [12289, 12289], [0, 20000]])
def test_logits_bias_lists_of_uneven_lengths(L, lists):  # noqa: F811
    """As many biased words as there are places for, one more, and many more, beside requests with few or none; histories and paths among them."""
    import torch
    V, R = 40000, len(lists)
    rng = np.random.default_rng(sum(lists))
    tokens = np.concatenate([rng.permutation(V)[:n] for n in lists]).astype(np.int32)
    values, off = rng.normal(0, 5, len(tokens)).astype(np.float32), np.concatenate([[0], np.cumsum(lists)])
    request = np.arange(3 * R) // 3
    history, drafted = rng.integers(0, V, (R, 900)).astype(np.int32), rng.integers(0, V, 3 * R).astype(np.int32)
    x = torch.randn((3 * R, V), device="cuda", generator=torch.Generator(device="cuda").manual_seed(R))
    want = x.double().cpu().numpy()
    for t, r in enumerate(request):
        count = np.bincount(np.concatenate([history[r], drafted[3 * r:t + 1]]), minlength=V)
        want[t] = np.where(count > 0, np.where(want[t] > 0, want[t] / 1.25, want[t] * 1.25), want[t]) - 0.125 * count
        want[t, tokens[off[r]:off[r + 1]]] += values[off[r]:off[r + 1]]
    policy = L.logits_policy_of(V, ints(history.reshape(-1)), ints(np.arange(R + 1) * 900), None, ints([1.25] * R, torch.float32), None, ints([0.125] * R, torch.float32),
                                ints(tokens), ints(values, torch.float32), ints(off))
    drafts, st = L.logits_drafts_of(ints(drafted), ints(request), ints(np.arange(R + 1) * 3)), L.Status()
    out = L.logits_edit(policy, drafts, x, st)
    assert st.read() == 0
    check_edit(out, want, list(request), out)
    L.logits_edit(policy, drafts, x, st, out=x)
    assert st.read() == 0 and torch.equal(x, out)


def test_logits_beside_out_in_one_buffer(L):  # noqa: F811
    """Rows of logits and of out that lie among one another without overlapping, with equal strides and different ones, and in place with a stride."""
    import torch
    V = 1000
    policy, drafts, st = L.logits_policy_of(V, ints([1, 1, 7]), ints([0, 3]), frequency=ints([0.5], torch.float32)), L.logits_drafts_of(row_request=ints([0] * 5)), L.Status()
    x = torch.randn((5, V), device="cuda")
    want = x.clone()
    want[:, 1] -= 1.0
    want[:, 7] -= 0.5
    def views(kind):
        flat = torch.full((60000,), 9.0, device="cuda")
        at = lambda start, stride: flat[start:].as_strided((5, V), (stride, 1), flat.storage_offset() + start)  # noqa: E731
        return {"pairs": (at(0, 2000), at(1000, 2000)), "pairs_back": (at(1000, 2000), at(0, 2000)), "far": (at(0, 1000), at(5000, 1000)),
                "threes": (at(0, 3000), at(2000, 6000)), "inside": (at(1000, 8000), at(2000, 1000)), "in_place": (at(3, 1234),) * 2}[kind]
    for kind in ("pairs", "pairs_back", "far", "threes", "inside", "in_place"):
        rows, out = views(kind)
        rows.copy_(x)
        L.logits_edit(policy, drafts, rows, st, out=out)
        assert st.read() == 0 and torch.equal(out, want), kind
        assert kind == "in_place" or torch.equal(rows, x), kind


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_logits_more_rows_than_a_grid_has(L, dtype):  # noqa: F811
    """70 000 rows of a small vocabulary, of 35 000 requests with a history of two words each; every seventh row is padding."""
    import torch
    rows, R, V = 70000, 35000, 37
    rng = np.random.default_rng(3)
    x = torch.tensor(rng.normal(0, 3, (rows, V)).astype(np.float32), device="cuda").to(getattr(torch, dtype))
    request = np.arange(rows) // 2
    request[::7] = -1
    history, frequency = rng.integers(0, V, (R, 2)).astype(np.int32), rng.uniform(0, 0.5, R).astype(np.float32)
    policy = L.logits_policy_of(V, ints(history.reshape(-1)), ints(np.arange(R + 1) * 2), frequency=ints(frequency, torch.float32))
    st, out = L.Status(), torch.full_like(x, 7.0)
    before = out.clone()
    L.logits_edit(policy, L.logits_drafts_of(row_request=ints(request)), x, st, out=out)
    assert st.read() == 0
    want, count = x.double().cpu().numpy(), np.zeros((R, V))
    np.add.at(count, (np.repeat(np.arange(R), 2), history.reshape(-1)), 1)
    want -= frequency[request][:, None].astype(np.float64) * count[request]
    check_edit(out, want, request, before)


def test_logits_captured_and_replayed_with_other_words(L):  # noqa: F811
    """Two graphs on two streams, replayed while histories, offsets, paths, masks and rows change; the results are those of calls one at a time."""
    import torch
    V, R, rows, most = 20000, 3, 9, 4000
    made = []
    for g in range(2):
        rng = np.random.default_rng(g)
        t = dict(history=ints([0] * most), offsets=ints([0] * (R + 1)), penalty=ints([1.0] * R, torch.float32), drafted=ints([0] * rows), request=ints([0] * rows),
                 begin=ints([0] * (R + 1)), ancestors=ints([0] * rows, torch.int64), grammar=ints([[0] * 625] * rows), x=torch.zeros((rows, V), device="cuda"))
        policy = L.logits_policy_of(V, t["history"], t["offsets"], None, t["penalty"], t["penalty"], t["penalty"])
        drafts, st, out, stream = L.logits_drafts_of(t["drafted"], t["request"], t["begin"], t["ancestors"], tree=True), L.Status(), torch.zeros((rows, V), device="cuda"), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            L.logits_edit(policy, drafts, t["x"], st, grammar=t["grammar"], out=out)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                L.logits_edit(policy, drafts, t["x"], st, grammar=t["grammar"], out=out)
        made.append((rng, t, policy, drafts, st, out, stream, graph))
    torch.cuda.synchronize()
    for st in (m[4] for m in made):
        st.reset()                                               # (the first call's rows lay outside their request)
    torch.cuda.synchronize()
    for fresh in ([4, 0, 5], [1, 1, 1], [0, 0, 9]):
        for rng, t, policy, drafts, st, out, stream, graph in made:
            with torch.cuda.stream(stream):
                n, history = sum(fresh), [int(h) for h in rng.integers(0, most // R, R)]
                at = np.concatenate([[0], np.cumsum(history)])
                new = dict(history=rng.integers(0, V, most), offsets=at, drafted=rng.integers(0, V, rows), begin=np.concatenate([[0], np.cumsum(fresh)]),
                           request=sum(([r] * f for r, f in enumerate(fresh)), []) + [-1] * (rows - n),
                           ancestors=[(1 << i) | 1 for f in fresh for i in range(f)] + [0] * (rows - n), grammar=rng.integers(-2 ** 31, 2 ** 31, (rows, 625)))
                for name, value in new.items():
                    t[name].copy_(ints(np.asarray(value).tolist(), t[name].dtype))
                t["penalty"].uniform_(0.5, 1.5)
                t["x"].normal_()
                out.fill_(7.0)
                graph.replay()
        torch.cuda.synchronize()
        for rng, t, policy, drafts, st, out, stream, graph in made:
            alone = torch.full_like(out, 7.0)
            assert st.read() == 0
            L.logits_edit(policy, drafts, t["x"], st, grammar=t["grammar"], out=alone)
            assert st.read() == 0 and torch.equal(out, alone) and bool((out[sum(fresh):] == 7.0).all())


# ---- plan: requests whose lengths are bad -----------------------------------------------------------------------------

@pytest.mark.parametrize("tree", [None, "random"])
@pytest.mark.parametrize("change", ["negative_cached", "fresh_above_its_bound", "sum_above_its_bound", "far"])
def test_plan_leaves_requests_with_bad_lengths_alone(L, change, tree):  # noqa: F811
    """Rows of a request with a negative length or one above its bound get no slot, and the request no pages and no table entries; the others
    are planned as if it brought no pages, and the rows behind it lie where its fresh tokens leave them."""
    import torch
    cached, fresh = [20, 30, 33], [3, 4, 5]
    s = Step(L, cached, fresh, 16, tree=tree, extra_tokens=9)
    s.step.longest_fresh, s.step.longest = 5, 38
    if change == "negative_cached":
        s.cached_dev[1] = -1
        n, position = 4, 0
    elif change == "fresh_above_its_bound":
        s.fresh_dev[1] = 6                                       # (and 30 + 6 is within `longest`)
        n, position = 6, 30
    elif change == "sum_above_its_bound":
        s.cached_dev[1] = 35                                     # 35 + 4: one more than `longest`
        n, position = 4, 35
    else:
        s.cached_dev[1] = 2 ** 31 - 1
        n, position = 4, 2 ** 31 - 1
    if tree:                                                     # parents of rows that moved: children of the cache
        s.step._keep[2][3:].fill_(-1)
    before = s.table_dev.clone()
    used = s.plan()
    assert s.status.read() == 2
    held = s.table
    want = [int(held[0, 1]) * 16 + 4 + i for i in range(3)] + [-1] * n
    free = s.free.tolist()
    # request 0 stays in its page; request 2 has 33 tokens in three pages: 34 .. 38 stay there too
    want += [int(held[2, 2]) * 16 + 1 + i for i in range(5)]
    want += [-1] * (s.tokens - len(want))
    assert s.step.slots_tensor.tolist() == want
    assert s.step.offsets_tensor.tolist() == [0, 3, 3 + n, 8 + n] and used.tolist() == [0]
    assert s.step.row_request_tensor.tolist() == [0] * 3 + [1] * n + [2] * 5 + [-1] * (s.tokens - 8 - n)
    assert torch.equal(s.table_dev, before) and free == s.free_dev.tolist()
    if not tree:
        assert s.step.positions_tensor.tolist()[3:3 + n] == [min(position + i, 2 ** 31 - 1) for i in range(n)]


def test_plan_counts_pages_of_good_requests_only(L):  # noqa: F811
    """Pages of the requests around a bad one are those that they would get without it."""
    for bad in ([-7, 4], [60, 5], [10, 60]):
        s = Step(L, [14, 10, 30, 1], [4, 5, 4, 3], 16, extra_tokens=60)
        s.step.longest_fresh, s.step.longest = 5, 64
        free = s.free.tolist()
        s.cached_dev[1], s.fresh_dev[1] = bad
        used = s.plan()
        assert s.status.read() == 2 and used.tolist() == [2]
        table, f = s.table_dev.cpu().numpy(), bad[1]
        assert [table[0, 1], table[2, 2]] == free[:2]
        slots = s.step.slots_tensor.tolist()
        assert slots[4:4 + f] == [-1] * f
        page = lambda r, n: int(table[r, n // 16]) * 16 + n % 16  # noqa: E731
        assert slots[:4] == [page(0, 14 + i) for i in range(4)] and slots[4 + f:8 + f] == [page(2, 30 + i) for i in range(4)]
        assert slots[8 + f:11 + f] == [page(3, 1 + i) for i in range(3)]


# ---- attention: weights far below the largest -------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("group", [2, 12])
@pytest.mark.parametrize("above", [8, 12, 15, 16, 17, 20])
def test_attention_one_key_far_above_the_others(L, above, group, dtype):  # noqa: F811
    """A key (one for each 16 of a block of 64) whose score is `above` nats over two thousand others and whose value is zero: what is left is the
    others' weights, e^-above each, which f16 would hold with few bits or none beside a weight of one. The bound counts half a
    step of every weight."""
    import torch
    s = Step(L, [2000] * 64, [1] * 64, 16)
    _, q, k, v, cache = attend(L, s, 8, group, 64, dtype)
    q.zero_()
    q[..., 0] = 1
    k.zero_()
    v.fill_(1000)
    for j in range(0, 64, 16):
        page = ints(s.table[:, j // 16]).long()
        k[page, :, j % 16, 0], v[page, :, j % 16] = above, 0
    out = torch.full_like(q, 7.0)
    L.attention_paged(cache, s.step, q, 1.0, s.status, out=out)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v, 1.0)


@pytest.mark.parametrize("fresh", [1, 40])
@pytest.mark.parametrize("scale", [1.1755e-38, 1e-30, 2.358e38])
def test_attention_smallest_and_largest_scales(L, scale, fresh):  # noqa: F811
    """At both ends of what is taken: every key has the same weight (with the largest scale, for queries of zero)."""
    import torch
    s = Step(L, [500, 3], [fresh, 2], 32)
    _, q, k, v, cache = attend(L, s, 2, 4, 128, "bfloat16")
    if scale > 1:
        q.zero_()
    out = torch.full_like(q, 7.0)
    L.attention_paged(cache, s.step, q, scale, s.status, out=out)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v, scale)


@pytest.mark.parametrize("fresh,dim,cached", [(1, 64, 300), (1, 128, 3000), (1, 256, 300), (20, 64, 300), (20, 128, 3000), (20, 256, 300)])
def test_attention_of_the_largest_values(L, fresh, dim, cached):  # noqa: F811
    """Values of 65504, or its negative, throughout, and keys whose weights all round up: a mean is never more than the largest value, so it is not
    infinite either."""
    import torch
    scores = np.unique(np.linspace(-0.9, -0.4, 1000).astype(np.float16))
    weights = np.exp(scores.astype(np.float64))
    up_most = scores[np.argsort(weights / weights.astype(np.float16).astype(np.float64))][:16]      # those that are rounded up by most
    for few in (False, True):                                    # items split over many CTAs, and whole ones
        s = Step(L, [cached] * (16 if few else 2), [fresh] * (16 if few else 2), 16)
        heads = 32 if few else 1
        _, q, k, v, cache = attend(L, s, heads, 2, dim, "float16")
        q.zero_()
        q[..., 0] = 1
        k.zero_()
        for r, x in enumerate(up_most[:len(s.cached)]):
            k[ints(s.table[r, :up(cached + fresh, 16)]).long(), :, :, 0] = float(x)
            k[int(s.table[r, 0]), :, 0, 0] = 0
        v.fill_(65504)
        v[:, :, :, dim // 2:] = -65504
        out = torch.full_like(q, 7.0)
        L.attention_paged(cache, s.step, q, 1.0, s.status, out=out)
        assert s.status.read() == 0
        check_attention(s, out, q, k, v, 1.0)


# ---- attention: more requests than a CTA counts at a time -------------------------------------------------------------

@pytest.mark.parametrize("requests,most,tree", [(127, 2, None), (128, 1, None), (129, 2, None), (300, 1, None), (1100, 2, None), (390, 20, None), (390, 40, "random"), (800, 20, "star"), (33, 140, None),
                                                (49, 140, None)])
@pytest.mark.parametrize("dtype,dim,group", [("bfloat16", 128, 2), ("float16", 256, 4), ("float16", 64, 3)])
def test_attention_of_more_requests_than_a_cta_has_threads(L, requests, most, tree, dtype, dim, group):  # noqa: F811
    """Lengths counted in several rounds, with bad ones among them (whose rows stay as they were) and long runs without fresh tokens."""
    import torch
    rng = np.random.default_rng(requests + most)
    fresh = (rng.integers(1, min(most, 6) + 1, requests) * (rng.random(requests) < 0.7)).tolist()
    for r in range(requests // 3, requests // 3 + requests // 5):
        fresh[r] = 0
    fresh[-1] = most
    cached = (300 * rng.random(requests) ** 3).astype(int).tolist()
    s = Step(L, cached, fresh, 16, seed=most, tree=tree)
    out, q, k, v, cache = attend(L, s, 2, group, dim, dtype, most)
    assert s.status.read() == 0
    check_attention(s, out, q, k, v)
    # a request whose cached tokens are more than there can be, in the middle
    bad = requests // 2 + requests // 8
    s.cached_dev[bad] = 1 << 20
    got = torch.full_like(out, 7.0)
    L.attention_paged(cache, s.step, q, dim ** -0.5, s.status, out=got)
    assert s.status.read() == 2
    b, e = s.want["offsets"][bad], s.want["offsets"][bad + 1]
    assert bool((got[b:e] == 7.0).all())
    got[b:e] = out[b:e]                                          # the others: as before, but for shares that are cut elsewhere
    check_attention(s, got, q, k, v)


@pytest.mark.parametrize("most", [1, 40])
def test_attention_of_a_step_without_fresh_tokens(L, most):  # noqa: F811
    """A captured step whose requests all wait: nothing is written and nothing reported."""
    s = Step(L, [30, 0, 100], [0, 0, 0], 16, extra_tokens=3)
    s.step.longest_fresh = most
    out, q, k, v, _ = attend(L, s, 2, 4, 128, "bfloat16")
    assert s.status.read() == 0 and bool((out == 7.0).all())


@pytest.mark.parametrize("fresh,tree", [(1, None), (4, None), (40, "random")])
def test_attention_of_pages_that_the_kernel_before_has_written_again(L, fresh, tree):  # noqa: F811
    """Pages, slots and queries are written anew before every attention, with nothing waited for between them: no call sees what an earlier
    one has read from the same places."""
    import torch
    def go(wait):
        s = Step(L, [500, 200], [fresh, fresh], 16, tree=tree)
        gen = torch.Generator(device="cuda").manual_seed(11)
        k, v = (torch.zeros((s.pages, 2, 16, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        cache, outs = L.kv_cache_of(k, v), []
        s.plan()
        tables = [s.table_dev.clone() for _ in range(2)]
        tables[1][:, :12] = s.table_dev[:, :12].flip(1)          # the same pages in another order
        every = torch.arange(s.pages * 16, device="cuda")
        ws, rows = L.attention_paged_workspace(cache, s.step, 8), torch.empty((s.pages * 16, 2, 2, 128), dtype=torch.bfloat16, device="cuda")
        q = torch.empty((s.tokens, 8, 128), dtype=torch.bfloat16, device="cuda")
        for i in range(24):
            rows.normal_(generator=gen)
            q.normal_(generator=gen)
            s.table_dev.copy_(tables[i % 2])
            slots = every.roll(i)
            L.kv_append(cache, slots, rows[:, 0], rows[:, 1], s.status)
            for _ in range(2):                                   # (the second call's kernels follow the first's)
                outs.append(L.attention_paged(cache, s.step, q, 0.1, s.status, workspace=ws))
            L.kv_append(cache, every, rows[:, 1], rows[:, 0], s.status)
            outs.append(L.attention_paged(cache, s.step, q, 0.1, s.status, workspace=ws))
            if wait:
                torch.cuda.synchronize()
        assert s.status.read() == 0
        return outs
    for a, b in zip(go(False), go(True)):
        assert torch.equal(a, b) and torch.isfinite(a).all()
