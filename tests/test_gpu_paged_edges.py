"""A serving step over a paged cache on a B200, at its edges: word lists that do not fit a table, requests whose lengths are bad, weights far
below the largest, against plain restatements in 64 bits."""
import numpy as np
import pytest

import paged_oracle as O
from test_gpu_paged import L, Step, check_attention, check_edit, ints, up  # noqa: F401

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
