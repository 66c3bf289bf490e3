"""Tokens sorted by expert, and the experts' rows, restated in plain loops and 64 bits for the tests."""

import torch


def plan_rows(T, k, E, align):
    n = T * k
    return (n + min(E, n) * (align - 1)) // align * align


def sort(ids, E, align):
    """(sources, positions, offsets, counts) as Python lists, from the definition."""
    T, k = ids.shape
    rows = [[] for _ in range(E)]
    for i, e in enumerate(ids.reshape(-1).tolist()):
        if 0 <= e < E:
            rows[e].append(i)
    sources, positions, offsets = [-1] * plan_rows(T, k, E, align), [-1] * (T * k), [0]
    for own in rows:
        for j, i in enumerate(own):
            sources[offsets[-1] + j] = i
            positions[i] = offsets[-1] + j
        offsets.append(offsets[-1] + -(-len(own) // align) * align)
    return sources, positions, offsets, [len(own) for own in rows]


def choices(T, k, E, seed, drop=0.0, dtype=torch.int32):
    """k choices a token, some the same, some absent (below zero and above E)."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, E, (T, k), generator=g)
    gone = torch.rand(T, k, generator=g)
    ids = torch.where(gone < drop / 2, torch.full_like(ids, -1), ids)
    return torch.where(gone > 1 - drop / 2, ids + E, ids).to(dtype)


def permute(x, sources, k):
    """float64 [R, H]."""
    src = torch.tensor(sources, dtype=torch.long)
    out = torch.zeros(len(sources), x.shape[1], dtype=torch.float64)
    made = src >= 0
    out[made] = x.double()[src[made] // k]
    return out


def gather(rows, positions, T, k):
    """float64 [T, k, H]: the rows of each choice, zeros for absent ones."""
    pos = torch.tensor(positions, dtype=torch.long)
    out = torch.zeros(T * k, rows.shape[1], dtype=torch.float64)
    made = pos >= 0
    out[made] = rows.double()[pos[made]]
    return out.reshape(T, k, rows.shape[1])
