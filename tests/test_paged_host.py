"""What the entries of a serving step refuse before any launch, and the description structs (no GPU)."""
import ctypes as C
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, NOMEM, UNSUPPORTED, BOUNDS, INVALID = 0, -2, -5, -7, -10
P = 0x10000                                                      # an aligned address that is never read


@pytest.fixture(scope="module")
def L():
    from yvex_b200 import build
    build.build()
    from yvex_b200 import lib
    return lib


def cache(L, **change):
    c = L.KvCache(30, 100, 16, 2, 128, P, P)
    for n, x in change.items():
        setattr(c, n, x)
    return c


def step(L, **change):
    s = L.KvStep(3, 12, 5, 4, 80, 0, P, P, P, P, P, P, P, P, P)
    for n, x in change.items():
        setattr(s, n, x)
    return s


def plan(L, c=None, s=None, free=P, count=9, used=P, status=P):
    return L.lib.yvex_b200_kv_plan(c or cache(L), s or step(L), free, count, used, status, None)


def append(L, c=None, slots=P, tokens=4, qtype=0, k=P, ks=256, v=P, vs=256, status=P):
    return L.lib.yvex_b200_kv_append(c or cache(L), slots, tokens, qtype, k, ks, v, vs, status, None)


def attend(L, c=None, s=None, q=P, stride=1024, heads=8, scale=0.1, out=P, ws=P, ws_bytes=1 << 40, status=P):
    return L.lib.yvex_b200_attention_paged(c or cache(L), s or step(L), q, stride, heads, scale, out, ws, ws_bytes, status, None)


def edit(L, p=None, d=None, qtype=0, x=P, xs=1000, g=P, gs=32, out=P, os_=1000, status=P):
    return L.lib.yvex_b200_logits_edit(p or L.LogitsPolicy(1000, 3), d or L.LogitsDrafts(3), qtype, x, xs, g, gs, out, os_, status, None)


SIZES = [("requests", 0, INVALID), ("tokens", 0, INVALID), ("table_width", 0, INVALID), ("longest_fresh", 0, INVALID), ("longest", 0, INVALID),
         ("longest_fresh", 81, BOUNDS), ("requests", 1 << 31, BOUNDS), ("tokens", 1 << 31, BOUNDS), ("longest", (1 << 30) + 1, BOUNDS), ("table_width", 1 << 32, BOUNDS)]


@pytest.mark.parametrize("name,value,code", SIZES)
def test_steps_that_are_refused(L, name, value, code):
    before = L.lib.yvex_b200_launch_count()
    assert plan(L, s=step(L, **{name: value})) == code
    assert attend(L, s=step(L, **{name: value})) == code
    assert L.lib.yvex_b200_attention_paged_workspace_bytes(cache(L), step(L, **{name: value}), 8) == 0
    assert L.lib.yvex_b200_launch_count() == before


CACHES = [("qtype", 0, UNSUPPORTED), ("qtype", 8, UNSUPPORTED), ("head_dim", 96, UNSUPPORTED), ("head_dim", 512, UNSUPPORTED), ("page_size", 8, UNSUPPORTED),
          ("page_size", 24, UNSUPPORTED), ("page_size", 0, UNSUPPORTED), ("page_size", 1 << 30, BOUNDS), ("pages", 0, INVALID), ("pages", 1 << 32, BOUNDS),
          ("kv_heads", 0, INVALID), ("kv_heads", 4096, BOUNDS), ("k", None, INVALID), ("v", None, INVALID), ("k", P + 8, INVALID), ("v", P + 2, INVALID)]


@pytest.mark.parametrize("name,value,code", CACHES)
def test_caches_that_are_refused(L, name, value, code):
    before = L.lib.yvex_b200_launch_count()
    assert append(L, c=cache(L, **{name: value})) == code
    assert attend(L, c=cache(L, **{name: value})) == code
    assert L.lib.yvex_b200_launch_count() == before


def test_plan_refuses_before_launch(L):
    before = L.lib.yvex_b200_launch_count()
    for name in ("cached", "fresh", "block_table", "offsets", "slots", "positions", "row_request"):
        assert plan(L, s=step(L, **{name: None})) == INVALID
    for name in ("parents", "ancestors"):
        assert plan(L, s=step(L, tree=1, **{name: None})) == INVALID
    assert plan(L, free=None) == INVALID and plan(L, used=None) == INVALID and plan(L, status=None) == INVALID
    assert plan(L, c=cache(L, pages=0)) == INVALID and plan(L, c=cache(L, page_size=0)) == INVALID and plan(L, c=cache(L, page_size=1 << 25)) == BOUNDS
    assert plan(L, s=step(L, tree=1, longest_fresh=65)) == BOUNDS
    assert L.lib.yvex_b200_kv_plan(None, step(L), P, 1, P, P, None) == INVALID and L.lib.yvex_b200_kv_plan(cache(L), None, P, 1, P, P, None) == INVALID
    assert L.lib.yvex_b200_launch_count() == before


def test_append_refuses_before_launch(L):
    before = L.lib.yvex_b200_launch_count()
    for name in ("slots", "k", "v", "status"):
        assert append(L, **{name: None}) == INVALID
    assert append(L, tokens=0) == INVALID and append(L, tokens=1 << 31) == BOUNDS
    assert append(L, qtype=8) == UNSUPPORTED and append(L, ks=255) == BOUNDS and append(L, vs=0) == BOUNDS
    assert append(L, k=P + 4) == INVALID and append(L, v=P + 8) == INVALID and append(L, ks=258) == INVALID and append(L, qtype=1, vs=260) == INVALID
    assert L.lib.yvex_b200_launch_count() == before


def test_attention_refuses_before_launch(L):
    before = L.lib.yvex_b200_launch_count()
    need = L.lib.yvex_b200_attention_paged_workspace_bytes(cache(L), step(L), 8)
    assert need > 0 and need % 16 == 0
    assert attend(L, ws_bytes=need - 1) == NOMEM and attend(L, ws=None) == NOMEM and attend(L, ws=P + 8) == INVALID
    for name in ("q", "out", "status"):
        assert attend(L, **{name: None}) == INVALID
    for name in ("cached", "offsets", "block_table"):
        assert attend(L, s=step(L, **{name: None})) == INVALID
    assert attend(L, s=step(L, tree=1, ancestors=None)) == INVALID
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attend(L, scale=scale) == INVALID
    assert attend(L, heads=7) == INVALID and attend(L, heads=0) == INVALID and attend(L, heads=1 << 20, stride=1 << 30) == BOUNDS
    for pages, heads, size in ((1 << 20, 2, 1024), (1 << 30, 1024, 1 << 24), ((1 << 31) - 1, 2, 16)):      # rows that a 32-bit coordinate cannot name
        assert attend(L, c=cache(L, pages=pages, kv_heads=heads, page_size=size), heads=heads, stride=1 << 20) == BOUNDS
    assert attend(L, stride=1023) == BOUNDS and attend(L, stride=1028) == INVALID and attend(L, q=P + 8) == INVALID and attend(L, out=P + 2) == INVALID
    assert L.lib.yvex_b200_launch_count() == before


def test_logits_refuse_before_launch(L):
    before = L.lib.yvex_b200_launch_count()
    for name in ("x", "out", "status"):
        assert edit(L, **{name: None}) == INVALID
    assert edit(L, qtype=8) == UNSUPPORTED and edit(L, xs=999) == BOUNDS and edit(L, os_=0) == BOUNDS and edit(L, gs=31) == BOUNDS
    assert edit(L, x=P + 2) == INVALID and edit(L, qtype=1, out=P + 1) == INVALID and edit(L, g=P + 2) == INVALID
    for p, code in ((L.LogitsPolicy(0, 3), INVALID), (L.LogitsPolicy(1000, 0), INVALID), (L.LogitsPolicy(1 << 32, 3), BOUNDS), (L.LogitsPolicy(1000, 1 << 31), BOUNDS),
                    (L.LogitsPolicy(1000, 3, 9, 9, P), INVALID), (L.LogitsPolicy(1000, 3, 9, 9, None, None, None, None, None, None, P, None, P), INVALID),
                    (L.LogitsPolicy(1000, 3, 9, 9, None, None, None, None, None, None, P, P, None), INVALID), (L.LogitsPolicy(1000, 2), BOUNDS),
                    (L.LogitsPolicy(1000, 3, 1 << 31), BOUNDS), (L.LogitsPolicy(1000, 3, 0, 1 << 31), BOUNDS)):
        assert edit(L, p=p) == code
    for d, code in ((L.LogitsDrafts(0), INVALID), (L.LogitsDrafts(1 << 31), BOUNDS), (L.LogitsDrafts(3, 0, P, None, P), INVALID),
                    (L.LogitsDrafts(3, 0, P, P, None), INVALID), (L.LogitsDrafts(3, 1, P, P, P, None), INVALID)):
        assert edit(L, d=d) == code
    assert L.lib.yvex_b200_launch_count() == before


def test_python_front_end_refuses_what_it_can_see(L, monkeypatch):
    """Shapes, types, strides and devices are checked before the library is entered (host tensors stand in for a device's)."""
    import torch
    from types import SimpleNamespace as N
    monkeypatch.setattr(L, "_torch", lambda: torch)
    monkeypatch.setattr(L, "_device", lambda: -1)                # where a host tensor says it is
    monkeypatch.setattr(L, "_on", lambda dev: None)
    called = []
    monkeypatch.setattr(L, "lib", N(yvex_b200_kv_append=lambda *a: called.append(a) or 0, yvex_b200_kv_plan=lambda *a: called.append(a) or 0,
                                    yvex_b200_attention_paged=lambda *a: called.append(a) or 0, yvex_b200_logits_edit=lambda *a: called.append(a) or 0))
    i32, st = lambda *shape: torch.zeros(shape, dtype=torch.int32), N(word=torch.zeros(1, dtype=torch.int32))  # noqa: E731
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    for bad in ((k, k.half()), (k, k[:3]), (k[0], k[0]), (k.transpose(0, 1), k.transpose(0, 1)), (k.float(), k.double())):
        with pytest.raises(L.YvexError):
            L.kv_cache_of(*bad)
    c = L.kv_cache_of(k, k)
    assert (c.qtype, c.pages, c.kv_heads, c.page_size, c.head_dim) == (30, 4, 2, 16, 64)
    good = dict(cached=i32(3), fresh=i32(3), block_table=i32(3, 5), tokens=7, longest_fresh=3, longest=50)
    s = L.kv_step_of(**good)
    assert (s.requests, s.tokens, s.table_width, s.tree, s.parents, s.ancestors) == (3, 7, 5, 0, None, None)
    for n, x in (("cached", torch.zeros(3)), ("fresh", i32(2)), ("block_table", i32(2, 5)), ("block_table", i32(5, 3).T), ("parents", i32(6)), ("offsets", i32(3)),
                 ("slots", i32(7)), ("positions", i32(6)), ("cached", i32(6)[::2])):
        with pytest.raises(L.YvexError):
            L.kv_step_of(**dict(good, **{n: x}))
    rows, slots = torch.zeros((7, 2, 2, 64)), torch.zeros(7, dtype=torch.int64)
    L.kv_append(c, slots, rows[:, 0], rows[:, 1], st)
    assert called.pop()[5] == 256                                # the stride of a row of [k | v]
    for bad in ((slots[:6], rows[:, 0], rows[:, 1]), (slots, rows[:, 0], rows[:, 1].half()), (slots.int(), rows[:, 0], rows[:, 1]),
                (slots, rows[:, 0].transpose(1, 2), rows[:, 1].transpose(1, 2)), (slots, rows[:, 0, :, ::2], rows[:, 1, :, ::2]), (slots, rows[:, 0].double(), rows[:, 1].double())):
        with pytest.raises(L.YvexError):
            L.kv_append(c, *bad, st)
    q, ws = torch.zeros((7, 8, 64), dtype=torch.bfloat16), torch.zeros(64, dtype=torch.uint8)
    L.attention_paged(c, s, q, 0.1, st, workspace=ws)
    called.pop()
    for bad, more in ((q[:6], {}), (q.half(), {}), (q[:, :, :32], {}), (q, dict(out=q[:6])), (q, dict(out=q.float())), (q.transpose(0, 1), {}), (q, dict(workspace=ws.int()))):
        with pytest.raises(L.YvexError):
            L.attention_paged(c, s, bad, 0.1, st, **dict(dict(workspace=ws), **more))
    with pytest.raises(L.YvexError):
        L.kv_plan(c, s, torch.zeros(3), st)
    p, d, x = L.logits_policy_of(100, requests=3), L.logits_drafts_of(rows=3), torch.zeros((3, 100))
    L.logits_edit(p, d, x, st, grammar=i32(3, 4))
    called.pop()
    for bad, more in ((x[:2], {}), (x[:, :99], {}), (x.double(), {}), (torch.zeros((100, 3)).T, {}), (x, dict(out=x.half())), (x, dict(grammar=torch.zeros((3, 4)))), (x, dict(grammar=i32(2, 4)))):
        with pytest.raises(L.YvexError):
            L.logits_edit(p, d, bad, st, **more)
    with pytest.raises(L.YvexError):
        L.logits_policy_of(100, i32(5), i32(3), requests=3)
    with pytest.raises(L.YvexError):
        L.logits_edit(p, L.logits_drafts_of(i32(3), i32(3), i32(3)), x, st)      # offsets of two requests
    with pytest.raises(L.YvexError):
        L.logits_policy_of(100)
    with pytest.raises(L.YvexError):
        L.logits_drafts_of(i32(3), i32(4))
    # tensors of another device than the current one
    monkeypatch.setattr(L, "_device", lambda: 0)
    for call in (lambda: L.kv_cache_of(k, k), lambda: L.kv_step_of(**good), lambda: L.kv_plan(c, s, i32(3), st, i32(1)), lambda: L.kv_append(c, slots, rows[:, 0], rows[:, 1], st),
                 lambda: L.attention_paged(c, s, q, 0.1, st, workspace=ws), lambda: L.logits_edit(p, d, x, st), lambda: L.logits_policy_of(9, i32(1), i32(2)),
                 lambda: L.logits_drafts_of(i32(3), i32(3))):
        with pytest.raises(L.YvexError):
            call()
    assert not called


def test_mirrors_have_the_headers_fields(L):
    """The ctypes structs list the header's fields in its order."""
    text = open(os.path.join(ROOT, "include", "yvex_b200_kernels.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, mirror in (("kv_cache", L.KvCache), ("kv_step", L.KvStep), ("logits_policy", L.LogitsPolicy), ("logits_drafts", L.LogitsDrafts)):
        body = re.search(r"typedef struct yvex_b200_%s \{(.*?)\}" % name, text, re.S).group(1)
        fields = [re.sub(r".*[ *]", "", f.strip()) for line in body.split(";") if line.strip() for f in line.split(",")]
        assert fields == [n for n, _ in mirror._fields_], name
    assert int(re.search(r"YVEX_B200_TREE_NODES (\d+)", text).group(1)) == L.TREE_NODES
    assert C.sizeof(L.KvStep) == 15 * 8
