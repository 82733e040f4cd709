"""The 4-bit KV cache in plain 64-bit arithmetic, from the definition in include/provekv_b200.h."""
import numpy as np

BLOCK = 16
SCALES = np.array([(c / 8 * 2.0 ** -14) if c < 8 else (1 + (c % 8) / 8) * 2.0 ** (c // 8 - 15) for c in range(0xDF)])


def half_even(x):
    return np.rint(x)


def scale_codes(amax):
    """Index of the scale nearest to amax / 7 (ties: even index); above the largest by more than half a step: -1."""
    ideal = np.asarray(amax, np.float64) / 7.0
    hi = np.clip(np.searchsorted(SCALES, ideal), 1, len(SCALES) - 1)
    up, down = SCALES[hi] - ideal, ideal - SCALES[hi - 1]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
    # the next scale would be 7680: at half way the tie goes to the even one, which is 0xDE
    return np.where(ideal > (7168 + 7680) / 2, -1, code)


def quantise(x):
    """[.., d] f64 -> (codes [.., d] 0..15, scale codes [.., d/16]); every block must be representable."""
    b = x.reshape(x.shape[:-1] + (-1, BLOCK)).astype(np.float64)
    sc = scale_codes(np.abs(b).max(-1))
    assert (sc >= 0).all()
    s = SCALES[sc][..., None]
    n = np.clip(half_even(np.divide(b, s, out=np.zeros_like(b), where=s > 0)), -8, 7) + 8
    return n.astype(np.uint8).reshape(x.shape), sc.astype(np.uint8)


def dequantise(codes, sc):
    return (codes.astype(np.float64) - 8) * np.repeat(SCALES[sc], BLOCK, -1)


def put_row(page, head, t, side, codes, sc, dim):
    """Writes one row's codes into a page's bytes [heads][atoms][18 dim]."""
    atom, i = page[head, t // 16], t % 16
    row = (codes[0::2] | (codes[1::2] << 4)).astype(np.uint8)
    if side and dim == 128 and i & 2:
        row = np.concatenate([row[32:], row[:32]])
    at = (8 * dim if side else 0) + i * dim // 2
    atom[at:at + dim // 2] = row
    at = (17 if side else 16) * dim + i * dim // 16
    atom[at:at + dim // 16] = sc


def get_row(page, head, t, side, dim):
    atom, i = page[head, t // 16], t % 16
    at = (8 * dim if side else 0) + i * dim // 2
    row = atom[at:at + dim // 2]
    if side and dim == 128 and i & 2:
        row = np.concatenate([row[32:], row[:32]])
    codes = np.empty(dim, np.uint8)
    codes[0::2], codes[1::2] = row & 15, row >> 4
    at = (17 if side else 16) * dim + i * dim // 16
    return codes, atom[at:at + dim // 16].copy()


def decode_all(pages, table, lens, dim):
    """[seqs][2][heads][longest][dim] f64 of every held token (zeros behind)."""
    heads, page_tokens = pages.shape[1], pages.shape[2] * 16
    out = np.zeros((len(lens), 2, heads, max(int(max(lens)), 1), dim))
    for s, n in enumerate(lens):
        for j in range(n):
            page = pages[table[s, j // page_tokens]]
            for h in range(heads):
                for side in range(2):
                    codes, sc = get_row(page, h, j % page_tokens, side, dim)
                    out[s, side, h, j] = dequantise(codes, np.minimum(sc, len(SCALES) - 1))
    return out


def fill(rng, n_seqs, heads, dim, page_tokens, lens, spread=0.5):
    """A pool with random pages (also where no token lies) holding random keys and values; returns pages, table and
    the values [seqs][2][heads][longest][dim] in f64."""
    max_pages = max(1, max(-(-int(n) // page_tokens) for n in lens)) + 1
    n_pages = n_seqs * max_pages + 2
    pages = rng.integers(0, 256, (n_pages, heads, page_tokens // 16, 18 * dim)).astype(np.uint8)
    table = rng.permutation(n_pages)[:n_seqs * max_pages].reshape(n_seqs, max_pages).astype(np.int32)
    longest = max(1, int(max(lens)))
    x = rng.standard_normal((n_seqs, 2, heads, longest, dim)) * rng.lognormal(0, spread, (1, 2, heads, 1, dim))
    codes, sc = quantise(x)
    values = dequantise(codes, sc)
    for s, n in enumerate(lens):
        for j in range(int(n)):
            page = pages[table[s, j // page_tokens]]
            for h in range(heads):
                for side in range(2):
                    put_row(page, h, j % page_tokens, side, codes[s, side, h, j], sc[s, side, h, j], dim)
        values[s, :, :, int(n):] = 0.0
        table[s, -(-int(n) // page_tokens):] = -1  # entries behind the last page are not read
    return pages, table, values


def visible(kpos, qpos, window, sinks):
    return (kpos <= qpos) & ((window == 0) | (qpos - kpos < window) | (kpos < sinks))


def attend(q, values, lens, ends, positions, group, scale, window, sinks, q_lens):
    """out, lse, mass added, and for the error bounds A = sum p |v|, D = scale sum |q| |k| (its largest over the
    row) and V = sum |v|."""
    S, n, HQ, d = q.shape
    out, A, V = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    lse = np.full((S, n, HQ), -np.inf)
    D = np.zeros((S, n, HQ))
    mass = np.zeros((S, values.shape[2], values.shape[3]))
    for s in range(S):
        L = int(lens[s])
        for i in range(int(q_lens[s])):
            qpos = int(ends[s]) - int(q_lens[s]) + i
            for h in range(HQ):
                kv = h // group
                kpos = positions[s, kv, :L] if positions is not None else np.arange(L)
                see = visible(kpos, qpos, window, sinks)
                if not see.any():
                    continue
                k, v = values[s, 0, kv, :L][see], values[s, 1, kv, :L][see]
                x = scale * (k @ q[s, i, h])
                m = x.max()
                p = np.exp(x - m)
                lse[s, i, h] = m + np.log(p.sum())
                p /= p.sum()
                out[s, i, h] = p @ v
                A[s, i, h] = p @ np.abs(v)
                V[s, i, h] = np.abs(v).sum(0)
                D[s, i, h] = abs(scale) * (np.abs(k) @ np.abs(q[s, i, h])).max()
                mass[s, kv, np.flatnonzero(see)] += p
    return out, lse, mass, A, D, V


def evict(positions, mass, n, end, budget, sinks, recent):
    """(destination, source) slots of one head's moves, in order."""
    if n <= budget:
        return []
    m = np.where(mass[:n] > 0, mass[:n], 0.0)
    stays = (positions[:n] < sinks) | (positions[:n] >= end - recent)
    order = sorted(range(n), key=lambda j: (not stays[j], -m[j] if not stays[j] else 0.0, j))
    kept = np.zeros(n, bool)
    kept[order[:budget]] = True
    return list(zip(np.flatnonzero(~kept[:budget]).tolist(), (budget + np.flatnonzero(kept[budget:])).tolist()))
