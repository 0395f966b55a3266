"""Plain restatements, in python integers and 64-bit floats, of what a serving step over a paged cache computes."""
import numpy as np
import torch


def parents_of(rng, fresh, shape="random"):
    """One tree per request: parents as indexes among the request's own rows, -1 for children of the cache."""
    out = []
    for f in fresh:
        for i in range(f):
            if i == 0:
                out.append(-1)
            elif shape == "chain":
                out.append(i - 1)
            elif shape == "star":
                out.append(-1)
            else:
                out.append(int(rng.integers(-1, i)))
    return out


def plan(cached, fresh, table, free, page, tokens, parents=None):
    """The step's arrays for lengths, a table (numpy, changed in place) and free pages that are in order."""
    offsets, slots, positions, requests, masks = [0], [-1] * tokens, [0] * tokens, [-1] * tokens, [0] * tokens
    taken = 0
    for r, (c, f) in enumerate(zip(cached, fresh)):
        for p in range(-(-c // page), -(-(c + f) // page)):
            table[r, p] = free[taken]
            taken += 1
        for i in range(f):
            t, at = offsets[-1] + i, c + i
            slots[t] = int(table[r, at // page]) * page + at % page
            requests[t] = r
            depth = i
            if parents is not None:
                mask, up = 1 << i, parents[t]
                while up != -1:
                    mask |= 1 << up
                    up = parents[offsets[-1] + up]
                masks[t], depth = mask, bin(mask).count("1") - 1
            positions[t] = c + depth
        offsets.append(offsets[-1] + f)
    return dict(offsets=offsets, slots=slots, positions=positions, row_request=requests, ancestors=masks, taken=taken)


def signed(mask):
    """A 64-bit mask as torch holds it."""
    return mask - (1 << 64) if mask >= 1 << 63 else mask


def attention(q, k, v, table, cached, offsets, ancestors, scale):
    """q [tokens, Hq, D], k/v [pages, Hkv, S, D] on any device; ancestors: list of masks or None (chain). Returns (out, spread, score):
    the result, the weights' mean of |v| and the largest sum of |q k| scale per row, all [tokens, Hq, ...] in 64 bits; rows that see
    nothing are zero."""
    S, D, H = k.shape[2], k.shape[3], k.shape[1]
    G = q.shape[1] // H
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    spread, score = torch.zeros_like(out), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for r, c in enumerate(cached):
        b, e = offsets[r], offsets[r + 1]
        f = e - b
        n = c + f
        if not f or not n:
            continue
        at = torch.arange(n, device=q.device)
        pages = torch.as_tensor(np.asarray(table[r]), device=q.device).long()[at // S]
        kk, vv = (x[pages, :, at % S].double().transpose(0, 1) for x in (k, v))          # [H, n, D]
        sees = torch.zeros((f, n), dtype=torch.bool, device=q.device)
        sees[:, :c] = True
        for i in range(f):
            for j in range(f):
                sees[i, c + j] = j <= i if ancestors is None else bool(ancestors[b + i] >> j & 1)
        qq = q[b:e].double().reshape(f, H, G, D).permute(1, 0, 2, 3).reshape(H, f * G, D)
        seen = sees[:, None, :].expand(f, G, n).reshape(f * G, n)
        s = (qq @ kk.transpose(1, 2) * scale).masked_fill(~seen, -np.inf)
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(top == -np.inf, torch.zeros_like(top), top))
        total = w.sum(-1, keepdim=True)
        total = torch.where(total == 0, torch.ones_like(total), total)
        lay = lambda x: x.reshape(H, f, G, -1).permute(1, 0, 2, 3).reshape(f, H * G, -1)  # noqa: E731
        out[b:e], spread[b:e] = lay(w @ vv / total), lay(w @ vv.abs() / total)
        score[b:e] = lay((qq.abs() @ kk.abs().transpose(1, 2) * scale).masked_fill(~seen, 0.0).amax(-1, keepdim=True))[..., 0]
    return out, spread, score


def attention_bound(dtype, out, spread, score, keys, D):
    """How far an output in `dtype` may be off. Half a step of the result; every weight rounded once to `dtype` (half a step of it, so of
    the weights' mean of |v|); a score is a sum of D products in f32 (D half-steps of the sum of |q k|, which is the relative error of its
    weight, and a few steps of the exponential's argument, of at most that size, and of its result); weights and products are summed in f32, in any order, numerator and denominator."""
    u, f = torch.finfo(dtype).eps / 2, torch.finfo(torch.float32).eps / 2
    weight = f * ((D + 8) * score[..., None] + 8)
    return u * out.abs() + 1.01 * spread * (u + 2 * weight + 2 * f * keys) + torch.finfo(dtype).tiny


def logits(rows, request_of, history, prompt, repetition, presence, frequency, biases, paths, grammar, vocabulary):
    """rows [n, V] (f64 numpy) edited: history, biases [(word, value)], ... per request, paths and grammar words per row."""
    out = rows.astype(np.float64).copy()
    for t, r in enumerate(request_of):
        if r < 0:
            continue
        count = np.zeros(vocabulary)
        seen = np.zeros(vocabulary, bool)
        for i, w in enumerate(history[r]):
            if w >= 0:
                seen[w] = True
                count[w] += i >= prompt[r]
        for w in paths[t]:
            if w >= 0:
                seen[w] = True
                count[w] += 1
        x = out[t]
        x = np.where(seen, np.where(x > 0, x / repetition[r], x * repetition[r]), x)
        x = x - frequency[r] * count - presence[r] * (count > 0)
        for w, value in dict(biases[r]).items():
            x[w] += value
        if grammar is not None:
            word = np.arange(vocabulary)
            x[(grammar[t][word // 32].astype(np.int64) >> (word % 32)) & 1 == 0] = -np.inf
        out[t] = x
    return out
