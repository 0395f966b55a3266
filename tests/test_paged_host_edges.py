"""The serving step's Python front end and refusals at their edges (no GPU)."""
import gc
import weakref
from types import SimpleNamespace as N

import pytest


@pytest.fixture(scope="module")
def L():
    from yvex_b200 import build
    build.build()
    from yvex_b200 import lib
    return lib


@pytest.fixture
def front(L, monkeypatch):
    """The front end over a library that takes every call, with host tensors standing in for a device's."""
    import torch
    monkeypatch.setattr(L, "_torch", lambda: torch)
    monkeypatch.setattr(L, "_device", lambda: -1)
    monkeypatch.setattr(L, "_on", lambda dev: None)
    monkeypatch.setattr(L, "lib", N(**{"yvex_b200_" + n: lambda *a: 0 for n in ("kv_plan", "kv_append", "attention_paged", "logits_edit")}))
    return L


def i32(*shape):
    import torch
    return torch.zeros(shape, dtype=torch.int32)


def status():
    return N(word=i32(1))


def cache_and_step(L):
    import torch
    k = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16)
    return L.kv_cache_of(k, k), L.kv_step_of(i32(3), i32(3), i32(3, 5), tokens=7, longest_fresh=3, longest=50)


def test_a_step_keeps_what_a_captured_call_writes(front):
    """A captured plan or attention goes on using the count and the workspace that it was given: they live as long as the step's description,
    also where the caller's names for them are used again."""
    import torch
    c, s = cache_and_step(front)
    used, ws, q = i32(1), torch.zeros(64, dtype=torch.uint8), torch.zeros((7, 8, 64), dtype=torch.bfloat16)
    front.kv_plan(c, s, i32(3), status(), used)
    front.attention_paged(c, s, q, 0.1, status(), workspace=ws)
    refs = [weakref.ref(used), weakref.ref(ws)]
    del used, ws
    gc.collect()
    assert all(r() is not None for r in refs)
    del s
    gc.collect()
    assert all(r() is None for r in refs)


def test_histories_that_a_counter_cannot_count_are_refused(L):
    """A word's counter has 31 bits, for what occurs in the history and on a path of drafted words."""
    P, before = 0x10000, L.lib.yvex_b200_launch_count()
    drafts = L.LogitsDrafts(9, 0, P, P, P)
    for tokens in (2 ** 31 - 9, 2 ** 31 - 1):
        policy = L.LogitsPolicy(1000, 9, tokens, 0, P, P)
        assert L.lib.yvex_b200_logits_edit(policy, drafts, 0, P, 1000, None, 0, P, 1000, P, None) == -7
    assert L.lib.yvex_b200_launch_count() == before


def overlap(L, rows, start, stride, out, out_stride, qtype=0, V=1000):
    return L.lib.yvex_b200_logits_edit(L.LogitsPolicy(V, rows), L.LogitsDrafts(rows), qtype, start, stride, None, 0, out, out_stride, 0x10000, None)


def test_logits_and_out_that_overlap_without_being_the_same_rows_are_refused(L):
    """Rows that another row's words are written into: the same start with another stride, shifted views, one row inside another."""
    P, before = 1 << 20, L.lib.yvex_b200_launch_count()
    for rows, start, stride, out, out_stride, qtype in (
            (2, P, 1000, P, 1004, 0), (2, P, 2000, P, 1000, 0), (1, P, 1000, P + 4, 1000, 0), (1, P + 16, 1000, P, 1000, 0), (3, P, 1000, P + 4000, 1000, 0),
            (3, P + 4000, 1000, P, 1000, 0), (3, P, 2000, P + 4 * 999, 2000, 0), (3, P, 2000, P + 4 * 1001, 2000, 0), (3, P + 4 * 2999, 2000, P, 2000, 0),
            (5, P, 2000, P + 4000, 3000, 0), (2, P, 1000, P + 2, 1000, 1), (1 << 20, P, 1000, P + 4 * 1000 * ((1 << 20) - 1), 1000, 0),
            (4, P, 1 << 40, P + (3 << 42) + 3996, 1 << 40, 0), (9, P, 1000, P + 4 * 8999, 5000, 0)):
        assert overlap(L, rows, start, stride, out, out_stride, qtype) == -10, (rows, start - P, stride, out - P, out_stride, qtype)
    assert L.lib.yvex_b200_launch_count() == before


def test_descriptions_of_another_device_are_refused(front, monkeypatch):
    """A cache, a step, a policy, drafts or a status made on one device and used while another one is current."""
    import torch

    class Far(torch.Tensor):                                     # says that it lies on device 3
        def get_device(self):
            return 3

    far = lambda t: t.as_subclass(Far)  # noqa: E731
    k, q, ws = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((7, 8, 64), dtype=torch.bfloat16), torch.zeros(64, dtype=torch.uint8)
    rows, slots, x = torch.zeros((7, 2, 2, 64)), torch.zeros(7, dtype=torch.int64), torch.zeros((3, 100))
    made = {}
    for device, on in ((-1, lambda t: t), (3, far)):
        monkeypatch.setattr(front, "_device", lambda device=device: device)
        i64 = lambda n: on(torch.zeros(n, dtype=torch.int64))  # noqa: E731
        made[device] = dict(cache=front.kv_cache_of(on(k), on(k)), geometry=front.kv_geometry_of(4, 16), status=N(word=on(i32(1))),
                            step=front.kv_step_of(on(i32(3)), on(i32(3)), on(i32(3, 5)), 7, 3, 50, offsets=on(i32(4)), slots=i64(7), positions=on(i32(7)), row_request=on(i32(7))),
                            policy=front.logits_policy_of(100, on(i32(5)), on(i32(4))), drafts=front.logits_drafts_of(row_request=on(i32(3))))
    monkeypatch.setattr(front, "_device", lambda: -1)
    calls = dict(plan=(lambda d: front.kv_plan(d["cache"], d["step"], i32(3), d["status"], i32(1)), ("step", "status")),
                 append=(lambda d: front.kv_append(d["cache"], slots, rows[:, 0], rows[:, 1], d["status"]), ("cache", "status")),
                 space=(lambda d: front.attention_paged(d["cache"], d["step"], q, 0.1, d["status"], workspace=ws), ("cache", "step", "status")),
                 edit=(lambda d: front.logits_edit(d["policy"], d["drafts"], x, d["status"]), ("policy", "drafts", "status")))
    for name, (call, parts) in calls.items():
        call(made[-1])
        for part in parts:
            with pytest.raises(front.YvexError):
                call(dict(made[-1], **{part: made[3][part]}))
    # a plan reads no more of a cache than its sizes, and descriptions without arrays belong to no device
    for part in ("geometry", "cache"):
        front.kv_plan(made[3][part], made[-1]["step"], i32(3), status(), i32(1))
    monkeypatch.setattr(front, "_device", lambda: 3)
    bare = front.logits_policy_of(100, requests=3), front.logits_drafts_of(rows=3)
    monkeypatch.setattr(front, "_device", lambda: -1)
    front.logits_edit(*bare, x, status())
    with pytest.raises(front.YvexError):
        front.attention_paged_workspace(made[3]["cache"], made[-1]["step"], 8)


def test_scales_that_f32_cannot_carry_are_refused(L):
    """A subnormal scale is zero where the exponentials are computed (and zero times the -inf of an unseen key is NaN), and one near the
    largest number is infinite once it is in powers of two."""
    P, before = 0x10000, L.lib.yvex_b200_launch_count()
    cache, step = L.KvCache(30, 100, 16, 2, 128, P, P), L.KvStep(3, 12, 5, 4, 80, 0, P, P, P, P, P, P, P, P, P)
    for scale in (1e-40, 1.1e-38, 1e-45, 2.4e38, 3.4e38):
        assert L.lib.yvex_b200_attention_paged(cache, step, P, 1024, 8, scale, P, P, 1 << 40, P, None) == -10
    assert L.lib.yvex_b200_launch_count() == before


def test_descriptions_filled_in_by_hand(front, monkeypatch):
    """The structs of the C header, without what the front end remembers beside them."""
    import torch
    P, called = 0x10000, []
    monkeypatch.setattr(front, "lib", N(yvex_b200_kv_plan=lambda *a: called.append(a) or 0, yvex_b200_attention_paged_workspace_bytes=lambda *a: called.append(a) or 64))
    monkeypatch.setattr(torch, "empty", lambda *a, **k: None)
    step = front.KvStep(3, 12, 5, 4, 80, 0, P, P, P, P, P, P, P, P, P)
    front.kv_plan(front.KvCache(30, 100, 16, 2, 128, P, P), step, i32(3), status(), i32(1))
    front.attention_paged_workspace(front.KvCache(30, 100, 16, 2, 128, P, P), step, 8)
    assert len(called) == 2
