"""The 4-bit KV cache on the GPU against plain 64-bit arithmetic (kv4ref): codes bit for bit, attention within bounds
derived below, evictions row for row."""
import numpy as np
import pytest

import kv4ref
import provekv_b200 as pk
from provekv_b200 import _lib as L
from provekv_b200 import kv4

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return getattr(torch, name)


def _dev(a, dtype=None):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


def _ints(a):
    import torch
    return _dev(np.asarray(a, np.int32), torch.int32)


def _empty_cache(n_seqs, heads, dim, page_tokens, max_pages, rng, lens, **kw):
    import torch
    pages = torch.from_numpy(rng.integers(0, 256, (n_seqs * max_pages + 1, heads, page_tokens // 16, 18 * dim)).astype(np.uint8)).cuda()
    table = torch.randperm(n_seqs * max_pages + 1)[:n_seqs * max_pages].view(n_seqs, max_pages).int().cuda()
    return kv4.Kv4Cache(pages, table, _ints(lens), **kw)


# -- append and read --------------------------------------------------------------------------------------------------
def _hard_rows(rng, n, dim, dtype):
    """Rows whose quotients sit on and beside ties, zero blocks, blocks below the smallest scale, large ones."""
    import torch
    x = rng.standard_normal((n, dim)) * np.exp(rng.uniform(-9, 6, (n, 1)))
    b = x.reshape(n, -1, 16)
    s = kv4ref.SCALES[rng.integers(24, 0xA0, b.shape[:2])]
    ties = (rng.integers(-8, 8, b.shape) + 0.5) * s[..., None]
    ties[..., 0] = 7 * s                                   # the block's scale is s itself
    b[:n // 2] = np.where(np.abs(ties) <= 7 * s[..., None], ties, 0.0)[:n // 2]
    b[n // 8] *= 1 + 2.0 ** -12
    b[n // 4] *= 1 - 2.0 ** -23
    b[-1] = 0.0
    b[-2] *= 1e-7
    b[-3] = rng.standard_normal(b[-3].shape) * 2.0 ** -16  # scales below 2^-14
    b[-4] *= 7e4 / max(1.0, np.abs(b[-4]).max()) * 0.7     # close to the largest scale
    b[-5, :, :] = 7 * 2.0 ** -14 * rng.choice([-1, 1, 0.5], b[-5].shape)
    amax = 3.5 * (kv4ref.SCALES[0x40] + kv4ref.SCALES[0x41])
    b[-6] = amax * rng.choice([1, -0.3, 0.7], b[-6].shape)  # amax / 7 half way between two scales
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim,heads,page", [(64, 3, 16), (128, 2, 64), (128, 1, 48)])
def test_append_writes_the_definition_and_read_gives_it_back(dtype, dim, heads, page):
    import torch
    rng = np.random.default_rng(dim + page)
    n, seqs = 37, 3
    lens, new = [37, 60, 45], [37, 20, 1]
    cache = _empty_cache(seqs, heads, dim, page, -(-64 // page) + 1, rng, lens)
    before = cache.pages.cpu().numpy().copy()
    k, v = (_hard_rows(rng, seqs * n * heads, dim, _dt(dtype)).view(seqs, n, heads, dim) for _ in range(2))
    cache.append(k.cuda(), v.cuda(), _ints(new))
    cache.check()
    want, table = before.copy(), cache.page_table.cpu().numpy()
    values = np.zeros((2, seqs, n, heads, dim))
    for s in range(seqs):
        for i in range(new[s]):
            slot = lens[s] - new[s] + i
            for h in range(heads):
                for side, x in enumerate((k, v)):
                    codes, sc = kv4ref.quantise(x[s, i, h].double().numpy())
                    kv4ref.put_row(want[table[s, slot // page]], h, slot % page, side, codes, sc, dim)
                    values[side, s, i, h] = kv4ref.dequantise(codes, sc)
    got = cache.pages.cpu().numpy()
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
    for t in (torch.float32, torch.float16, torch.bfloat16):
        for side, r in enumerate(cache.read(n, t, _ints(new))):
            assert r.dtype == t and np.array_equal(r.double().cpu().numpy(), values[side])
    # rows behind a sequence's last stay as they were in a given output
    out = torch.full((2, seqs, n, heads, dim), 5.0, device="cuda").unbind(0)
    cache.read(n, None, _ints(new), out)
    for side in range(2):
        for s in range(seqs):
            assert (out[side][s, new[s]:] == 5.0).all() and np.array_equal(out[side][s, :new[s]].double().cpu().numpy(), values[side, s, :new[s]])
    cache.check()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_append_takes_strided_rows_and_keeps_statistics(dtype):
    import torch
    rng = np.random.default_rng(5)
    seqs, heads, dim, page, n = 2, 4, 64, 32, 9
    lens, ends = [9, 40], [9, 100]
    pos = torch.full((seqs, heads, 64), -7, dtype=torch.int32, device="cuda")
    mass = torch.full((seqs, heads, 64), 3.0, device="cuda")
    cache = _empty_cache(seqs, heads, dim, page, 2, rng, lens, ends=_ints(ends), positions=pos, mass=mass)
    packed = _dev(rng.standard_normal((n, seqs, 3 * heads, dim)), _dt(dtype))  # token first, K, V and something else side by side
    k, v = packed[:, :, :heads].transpose(0, 1), packed[:, :, heads:2 * heads].transpose(0, 1)
    cache.append(k, v)
    cache.check()
    for side, got in enumerate(cache.read(n, _dt(dtype))):
        x = (k, v)[side].double().cpu().numpy()
        assert np.array_equal(got.double().cpu().numpy(), kv4ref.dequantise(*kv4ref.quantise(x)))
    for s in range(seqs):
        first = lens[s] - n
        assert (pos[s, :, first:lens[s]].cpu() == torch.arange(ends[s] - n, ends[s])).all()
        assert (mass[s, :, first:lens[s]] == 0).all()
        assert (pos[s, :, :first] == -7).all() and (pos[s, :, lens[s]:] == -7).all()
        assert (mass[s, :, :first] == 3).all() and (mass[s, :, lens[s]:] == 3).all()


def test_rows_that_cannot_be_stored_are_reported_and_become_zeros():
    import torch
    rng = np.random.default_rng(6)
    cache = _empty_cache(2, 3, 64, 16, 2, rng, [5, 7])
    k, v = (_dev(rng.standard_normal((2, 5, 3, 64)), torch.float32) for _ in range(2))
    v[1, 2, 1, 40] = float("inf")
    k[1, 4, 0, 3] = 7.0 * 7500
    v[0, 3, 2, 63] = float("nan")
    cache.append(k, v)
    with pytest.raises(pk.PkvError) as e:
        cache.check()
    assert (e.value.status, e.value.vector_index) == (L.VEC_NONFINITE_INPUT, ((0 * 5 + 3) * 3 + 2) * 2 + 1)
    cache.check()  # read and cleared
    gk, gv = cache.read(5)
    assert (gv[1, 2, 1] == 0).all() and (gk[1, 4, 0] == 0).all() and (gv[0, 3, 2] == 0).all()
    assert (gk[1, 2, 1] != 0).any() and (gv[1, 4, 0] != 0).any()
    k2, v2 = k.clone(), v.clone().nan_to_num(0, 0, 0)
    cache.append(k2, v2)
    with pytest.raises(pk.PkvError) as e:
        cache.check()
    assert (e.value.status, e.value.vector_index) == (L.VEC_NORM_RANGE, ((1 * 5 + 4) * 3 + 0) * 2)


def test_bad_lengths_and_pages_are_reported_and_skipped():
    import torch
    rng = np.random.default_rng(7)
    cache = _empty_cache(4, 2, 128, 16, 4, rng, [20, 65, -1, 30])
    cache.page_table[3, 1] = cache.pages.shape[0]
    cache.page_table[0, 0] = -5
    before = cache.pages.clone()
    x = _dev(rng.standard_normal((4, 20, 2, 128)), torch.bfloat16)
    cache.append(x, x)
    with pytest.raises(pk.PkvError) as e:
        cache.check()
    assert (e.value.status, e.value.vector_index) == (L.VEC_BAD_SEQUENCE, 0)
    changed = set((cache.pages != before).flatten(1).any(1).nonzero().flatten().tolist())
    assert changed == {int(cache.page_table[0, 1]), int(cache.page_table[3, 0])}
    q = _dev(rng.standard_normal((4, 1, 4, 128)), torch.bfloat16)
    out, lse = cache.attend(q)
    with pytest.raises(pk.PkvError) as e:
        cache.check()
    assert (e.value.status, e.value.vector_index) == (L.VEC_BAD_SEQUENCE, 0)
    assert (out[1] == 0).all() and (out[2] == 0).all() and torch.isinf(lse[1:3]).all()
    # the tokens of the good pages alone
    table, pages = cache.page_table.cpu().numpy(), cache.pages.cpu().numpy()
    val = kv4ref.decode_all(pages, table[:, 1:], [4, 0, 0, 0], 128)
    want, wlse, _, A, D, V = kv4ref.attend(q.double().cpu().numpy(), val, [4, 0, 0, 0], [4, 1, 1, 4], None, 2, 128 ** -0.5, 0, 0, [1, 1, 1, 1])
    _close(out[:1], lse[:1], want[:1], wlse[:1], A[:1], D[:1], V[:1])
    bad = _ints([1, 2, 0, -1])
    cache.lens.copy_(_ints([20, 20, 20, 20]))
    cache.page_table[0, 0], cache.page_table[3, 1] = 0, 0
    out, lse = torch.full_like(q, 9.0), torch.full((4, 1, 4), 9.0, device="cuda")
    cache.attend(q, q_lens=bad, out=out, lse=lse)
    with pytest.raises(pk.PkvError) as e:
        cache.check()
    assert (e.value.status, e.value.vector_index) == (L.VEC_BAD_SEQUENCE, 1)
    assert (out[0] != 9).any() and (out[1:] == 9).all() and (lse[1:] == 9).all()


# -- attention ------------------------------------------------------------------------------------------------------------
def _within(got, want, tol, what):
    off = np.abs(got - want) - tol
    if not (off <= 0).all():
        at = np.unravel_index(np.nanargmax(np.where(np.isnan(off), np.inf, off)), off.shape)
        raise AssertionError(f"{what} at {at}: {got[at]} is not {want[at]} within {np.broadcast_to(tol, off.shape)[at]}")


def _close(out, lse, want, wlse, A, D, V):
    """Scores are f32 sums of dim exact products in at most 2 dim / 16 steps of the tensor cores, each within 2^-22 of the
    largest partial sum, and three f32 roundings after: off by at most eps = 2^-18 D.  A weight is then within a
    factor exp(2 eps) (its own error and its sum's) of the true one, and enters the second product in binary16 (2^-11; f32
    queries: two terms, 2^-21).  So out is off by (w + 2 eps + 2^-18) A plus its own rounding.
    Binary16 ends at 2^-25 (half its last subnormal): weights are kept 2^7 and more times too large, so a key of whatever weight
    is also off by up to 2^-32 of the row's largest weight, which is below 1 after the division by the sum: 2^-32 sum |v|."""
    import torch
    w, unit = {torch.float32: (2.0 ** -21, 2.0 ** -24), torch.float16: (2.0 ** -11, 2.0 ** -11),
               torch.bfloat16: (2.0 ** -11, 2.0 ** -8)}[out.dtype]
    got, glse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    eps = 2.0 ** -18 * D[..., None]
    tol = (w + 2 * eps + 2.0 ** -18) * A + 2.0 ** -32 * V + unit * np.abs(want) + (2.0 ** -25 if out.dtype == torch.float16 else 0.0)
    _within(got, want, tol, "out")
    none = np.isinf(wlse)
    assert np.array_equal(none, np.isneginf(glse)) and not np.isnan(glse).any()
    _within(glse[~none], wlse[~none], (eps[..., 0] + 2.0 ** -22 * np.abs(wlse) + 2.0 ** -20)[~none], "lse")


def _attend_case(seed, dtype, dim, heads, group, page, lens, q_len, window, sinks, moved, accumulate, q_lens=None, max_len=0,
                 scale=None):
    import torch
    rng = np.random.default_rng(seed)
    S = len(lens)
    pages, table, values = kv4ref.fill(rng, S, heads, dim, page, lens)
    cap = table.shape[1] * page
    ends, pos = np.asarray(lens), None
    if moved:
        ends = np.asarray(lens) + rng.integers(0, 50, S)
        pos = np.zeros((S, heads, cap), np.int32)
        for s, n in enumerate(lens):
            for h in range(heads):
                pos[s, h, :n] = rng.permutation(int(ends[s]))[:n]
    mass = _dev(np.abs(rng.standard_normal((S, heads, cap))), torch.float32) if accumulate else None
    mass0 = mass.double().cpu().numpy() if accumulate else None
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints(lens), ends=_ints(ends) if moved else None,
                         positions=_ints(pos) if moved else None, mass=mass)
    q = _dev(rng.standard_normal((S, q_len, heads * group, dim)) * 2, _dt(dtype))
    ql = q_lens if q_lens is not None else [q_len] * S
    before = cache.pages.clone()
    out, lse = cache.attend(q, scale=scale, window=window, sinks=sinks, accumulate=accumulate, max_len=max_len,
                            q_lens=None if q_lens is None else _ints(q_lens))
    cache.check()
    assert torch.equal(before, cache.pages)
    want = kv4ref.attend(q.double().cpu().numpy(), values, lens, ends, pos, group, dim ** -0.5 if scale is None else scale, window, sinks, ql)
    for s in range(S):  # padding rows of a fresh output are zeros
        assert (out[s, ql[s]:] == 0).all() and (lse[s, ql[s]:] == 0).all()
        want[1][s, ql[s]:] = 0.0
    _close(out, lse, want[0], want[1], *want[3:])
    if accumulate:
        got = mass.double().cpu().numpy()
        full = mass0.copy()
        full[:, :, :values.shape[3]] += want[2]
        eps = 2.0 ** -18 * want[4].max() + 2.0 ** -22 * np.abs(want[1][~np.isinf(want[1])]).max(initial=0.0) + 2.0 ** -19
        _within(got, full, 2 * eps * (full - mass0) + 2.0 ** -23 * full, "mass")
        assert np.array_equal(got[full == mass0], mass0[full == mass0])  # what no query saw is untouched
    return cache, q, out, lse


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim,heads,group,page", [(64, 2, 7, 16), (128, 2, 4, 64), (64, 3, 1, 48), (128, 1, 12, 32)])
@pytest.mark.parametrize("lens", [[1], [0, 16, 17, 33], [31, 32, 200]])
def test_single_tokens(dtype, dim, heads, group, page, lens):
    _attend_case(dim + len(lens), dtype, dim, heads, group, page, lens, 1, 0, 0, False, False)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (40, 4), (33, 40), (500, 3), (5, 1000)])
@pytest.mark.parametrize("moved", [False, True])
def test_windows_and_sinks(dtype, window, sinks, moved):
    _attend_case(window + sinks, dtype, 128, 2, 3, 32, [0, 5, 77, 210], 1, window, sinks, moved, True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("q_len,group", [(2, 1), (3, 4), (5, 7), (33, 2), (40, 1)])
@pytest.mark.parametrize("window,sinks,moved", [(0, 0, False), (20, 3, False), (0, 0, True), (30, 2, True)])
def test_several_tokens_are_causal(dtype, dim, q_len, group, window, sinks, moved):
    _attend_case(q_len * group, dtype, dim, 2, group, 16, [40, 41, 131], q_len, window, sinks, moved, True)


def test_padded_queries_and_more_queries_than_tokens():
    # 3 of 6 rows are padding in the first sequence, none in the second, all in the third; the fourth has fewer tokens than queries
    _attend_case(3, "float16", 128, 2, 2, 16, [30, 6, 12, 4], 6, 0, 0, False, True, q_lens=[3, 6, 0, 5])
    _attend_case(4, "float32", 64, 2, 2, 16, [30, 6, 12, 4], 6, 3, 1, True, True, q_lens=[3, 6, 0, 4])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_long_rows_are_split_and_joined(dtype):
    _attend_case(11, dtype, 64, 1, 2, 128, [3001], 1, 0, 0, False, True)
    _attend_case(12, dtype, 128, 1, 9, 64, [700, 1500], 1, 0, 0, False, False)
    _attend_case(13, dtype, 128, 1, 2, 64, [1700], 4, 900, 70, False, True)
    # a bound that is too small only makes the last part longer
    _attend_case(14, dtype, 64, 1, 2, 64, [1700, 3], 1, 0, 0, False, True, max_len=600)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("page,moved,window,sinks", [(48, False, 0, 0), (16, True, 500, 30), (48, False, 1200, 100), (64, True, 0, 0)])
def test_rows_share_runs_whatever_their_lengths(dtype, page, moved, window, sinks):
    """More than 32 sequences, some empty, of lengths that cut units and pages anywhere; the longest decides that rows share runs."""
    rng = np.random.default_rng(page + window)
    lens = [1700, 0, 1] + rng.integers(1, 400, 34).tolist() + [1650]
    _attend_case(15, dtype, 64, 1, 3, page, lens, 1, window, sinks, moved, True)


def test_runs_skip_sequences_without_queries():
    lens = [1700, 1650, 30, 800, 64]
    _attend_case(16, "bfloat16", 128, 2, 2, 64, lens, 3, 0, 0, False, True, q_lens=[0, 2, 3, 0, 1])
    _attend_case(17, "float32", 64, 1, 9, 64, lens, 2, 0, 0, False, True, q_lens=[1, 0, 0, 2, 0])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-3])
@pytest.mark.parametrize("lens,q_len", [([45, 70], 1), ([1700], 1), ([90], 30)])
def test_scales_that_are_zero_negative_or_small(dtype, scale, lens, q_len):
    _attend_case(18, dtype, 64, 2, 2, 16, lens, q_len, 40, 3, False, True, scale=float(np.float32(scale)))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page,lens,q_len,group,window,sinks,moved", [(48, [700], 60, 2, 0, 0, False), (16, [1300, 5, 0], 20, 1, 300, 70, False),
                                                                      (64, [1100, 1024], 18, 1, 0, 0, True), (48, [640], 300, 1, 50, 0, True)])
def test_chunks_split_over_the_tokens(dim, page, lens, q_len, group, window, sinks, moved):
    _attend_case(19 + page, "bfloat16", dim, 1, group, page, lens, q_len, window, sinks, moved, True,
                 q_lens=[min(q_len, n + 2) for n in lens])


@pytest.mark.parametrize("dtype,q_len,group", [("bfloat16", 30, 2), ("float16", 150, 2), ("float32", 20, 1), ("bfloat16", 9, 4)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 20)])
def test_queries_over_a_cache_that_was_thinned_out(dtype, q_len, group, window, sinks):
    """Ascending positions with gaps, as an eviction leaves them: most units are seen by every row, the last by some."""
    import torch
    rng = np.random.default_rng(q_len)
    lens, ends = [700, 330], np.array([900, 345])
    pages, table, values = kv4ref.fill(rng, 2, 2, 64, 32, lens)
    cap = table.shape[1] * 32
    pos = np.full((2, 2, cap), -5, np.int32)  # behind the length: anything
    for s, n in enumerate(lens):
        for h in range(2):
            old = np.sort(rng.permutation(int(ends[s]) - q_len)[:n - q_len])
            pos[s, h, :n] = np.r_[old, np.arange(ends[s] - q_len, ends[s])]
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints(lens), ends=_ints(ends), positions=_ints(pos),
                         mass=torch.zeros((2, 2, cap), device="cuda"))
    q = _dev(rng.standard_normal((2, q_len, 2 * group, 64)), _dt(dtype))
    out, lse = cache.attend(q, window=window, sinks=sinks, accumulate=True)
    cache.check()
    want = kv4ref.attend(q.double().cpu().numpy(), values, lens, ends, pos, group, 64 ** -0.5, window, sinks, [q_len] * 2)
    _close(out, lse, want[0], want[1], *want[3:])
    # a weight is off by its score's error and its sum's, and rounded once a row
    got = cache.mass.double().cpu().numpy()[:, :, :want[2].shape[2]]
    eps = 2.0 ** -18 * want[4].max() + 2.0 ** -22 * np.abs(want[1]).max() + 2.0 ** -19
    _within(got, want[2], (2 * eps + 2.0 ** -24 * q_len * group) * want[2], "mass")


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("q_len,group,heads,n", [(17, 1, 2, 300), (12, 4, 1, 700), (7, 7, 1, 500), (64, 1, 1, 1700), (50, 1, 1, 2500)])
def test_rows_on_both_sides_of_a_tile(dtype, q_len, group, heads, n):
    """17, 48, 49, 64 and 50 query rows a kv head; the last two in many splits."""
    _attend_case(23 + q_len, dtype, 128, heads, group, 64, [n], q_len, 0, 0, False, True)
    _attend_case(24 + q_len, dtype, 64, heads, group, 16, [n, 3], q_len, 130, 7, True, False)


def test_pages_missing_from_a_chunk_and_from_a_long_row():
    import torch
    for q_len, n in ((20, 300), (1, 1700)):
        rng = np.random.default_rng(n)
        pages, table, values = kv4ref.fill(rng, 2, 1, 128, 16, [n, 40])
        table[0, 3], table[0, 9] = -1, pages.shape[0] + 7
        cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([n, 40]), mass=torch.zeros((2, 1, table.shape[1] * 16), device="cuda"))
        q = _dev(rng.standard_normal((2, q_len, 2, 128)), torch.float16)
        out, lse = cache.attend(q, accumulate=True)
        with pytest.raises(pk.PkvError) as e:
            cache.check()
        assert (e.value.status, e.value.vector_index) == (L.VEC_BAD_SEQUENCE, 0)
        gone = np.r_[48:64, 144:160]
        pos = np.tile(np.arange(n, dtype=np.int64), (2, 1, 1))
        pos[0, 0, gone] = 1 << 30  # beyond every query: not seen
        w = kv4ref.attend(q.double().cpu().numpy(), values, [n, 40], [n, 40], pos, 2, 128 ** -0.5, 0, 0, [q_len] * 2)
        _close(out, lse, w[0], w[1], *w[3:])
        assert (cache.mass[0, 0, 48:64] == 0).all() and (cache.mass[0, 0, 64:100] > 0).all()


def test_a_longer_query_chunk():
    _attend_case(21, "bfloat16", 128, 1, 4, 64, [300], 200, 0, 0, False, True)
    _attend_case(22, "float16", 64, 2, 2, 48, [150, 260], 130, 50, 5, False, False, q_lens=[130, 77])


def test_large_and_small_scales_of_queries():
    """Rows of q far from 1 in either direction keep their bits (a power of two per row)."""
    for dtype, f in (("float32", 1e20), ("float32", 1e-20), ("bfloat16", 1e-30), ("bfloat16", 1e15), ("float16", 1e-4)):
        import torch
        rng = np.random.default_rng(31)
        pages, table, values = kv4ref.fill(rng, 1, 1, 64, 16, [50])
        cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([50]))
        q = _dev(rng.standard_normal((1, 1, 2, 64)) * f, _dt(dtype))
        scale = 0.125 / f
        out, lse = cache.attend(q, scale=scale)
        s32 = float(np.float32(scale))
        want = kv4ref.attend(q.double().cpu().numpy(), values, [50], [50], None, 2, s32, 0, 0, [1])
        _close(out, lse, want[0], want[1], *want[3:])


def test_queries_that_are_not_finite_spoil_their_own_rows_only():
    import torch
    rng = np.random.default_rng(32)
    pages, table, _ = kv4ref.fill(rng, 2, 2, 128, 16, [50, 3000])
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([50, 3000]))
    q = _dev(rng.standard_normal((2, 1, 8, 128)), torch.bfloat16)
    clean, _ = cache.attend(q)
    q2 = q.clone()
    q2[0, 0, 3, 5] = float("nan")
    q2[1, 0, 6, 100] = float("inf")
    out, lse = cache.attend(q2)
    spoilt = torch.zeros((2, 1, 8), dtype=torch.bool, device="cuda")
    spoilt[0, 0, 3] = spoilt[1, 0, 6] = True
    assert torch.isnan(out[spoilt]).all() and torch.isnan(lse[spoilt]).all()
    assert torch.equal(out[~spoilt], clean[~spoilt])


def test_sequences_may_share_a_prefix_and_repeat_a_page():
    import torch
    rng = np.random.default_rng(33)
    pages, table, values = kv4ref.fill(rng, 2, 2, 64, 16, [64, 64])
    table[1, :2] = table[0, :2]
    table[1, 2] = table[0, 1]
    values[1, :, :, :32] = values[0, :, :, :32]
    values[1, :, :, 32:48] = values[0, :, :, 16:32]
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([64, 64]))
    q = _dev(rng.standard_normal((2, 1, 4, 64)), torch.float16)
    out, lse = cache.attend(q)
    want = kv4ref.attend(q.double().cpu().numpy(), values, [64, 64], [64, 64], None, 2, 0.125, 0, 0, [1, 1])
    _close(out, lse, want[0], want[1], *want[3:])


def test_strided_queries_and_outputs():
    import torch
    rng = np.random.default_rng(34)
    pages, table, values = kv4ref.fill(rng, 2, 2, 64, 16, [30, 55])
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([30, 55]))
    packed = _dev(rng.standard_normal((3, 2, 12, 64)), torch.float32)
    q = packed[:, :, 4:10].transpose(0, 1)
    room = torch.full((2, 6, 4, 72), 7.0, device="cuda")
    out = room[..., 4:68].transpose(1, 2)[:, :3]
    got, lse = cache.attend(q, out=out)
    assert got.data_ptr() == out.data_ptr()
    want = kv4ref.attend(q.double().cpu().numpy(), values, [30, 55], [30, 55], None, 3, 0.125, 0, 0, [3, 3])
    _close(out, lse, want[0], want[1], *want[3:])
    assert (room[..., :4] == 7).all() and (room[..., 68:] == 7).all() and (room[:, :, 3] == 7).all()


def test_what_would_wrap_or_overlap_is_refused():
    import torch
    rng = np.random.default_rng(41)
    pages, table, _ = kv4ref.fill(rng, 2, 2, 64, 16, [30, 55])
    cap = table.shape[1] * 16
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([30, 55]), positions=torch.zeros((2, 2, cap), dtype=torch.int32, device="cuda"),
                         mass=torch.zeros((2, 2, cap), device="cuda"))
    q = torch.zeros((2, 1, 4, 64), device="cuda")
    wide = (1 << 32) + 5
    for bad in (dict(window=wide), dict(sinks=wide), dict(max_len=wide), dict(window=-1), dict(out=q[:1].expand(2, 1, 4, 64))):
        with pytest.raises(ValueError):
            cache.attend(q, **bad)
    for bad in ((wide, 0, 0), (20, wide, 0), (20, 0, wide), (-1, 0, 0)):
        with pytest.raises(ValueError):
            cache.evict(bad[0], sinks=bad[1], recent=bad[2])
    k = torch.zeros((2, 1, 2, 64), device="cuda")
    with pytest.raises(ValueError):
        cache.read(1, out=(k, k[:, :, :1].expand(2, 1, 2, 64)))
    assert (cache.mass == 0).all() and (cache.pages.cpu().numpy() == pages).all()


def test_strides_of_dimensions_of_one_do_not_count():
    import torch
    rng = np.random.default_rng(42)
    pages, table, values = kv4ref.fill(rng, 1, 1, 64, 16, [30])
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([30]))
    q = _dev(rng.standard_normal(64), torch.float32).as_strided((1, 1, 1, 64), (1, 3, 5, 1))
    out, lse = cache.attend(q)
    want = kv4ref.attend(q.double().cpu().numpy(), values, [30], [30], None, 1, 0.125, 0, 0, [1])
    _close(out, lse, want[0], want[1], *want[3:])


@pytest.mark.parametrize("dtype,q_len", [("float32", 6), ("bfloat16", 6), ("bfloat16", 70)])
def test_the_widest_window_with_more_queries_than_tokens(dtype, q_len):
    # positions below zero minus the window do not fit 32 bits
    _attend_case(43, dtype, 64, 1, 2, 16, [4, 66], q_len, (1 << 31) - 1, 0, False, True)
    _attend_case(44, dtype, 64, 1, 2, 16, [4, 66], q_len, (1 << 31) - 1, 2, True, True)


def test_ends_below_the_lengths_read_and_write_nothing_else():
    """Ends that were never raised: whatever the queries see, no row before the first is read and mass stays finite."""
    import torch
    rng = np.random.default_rng(45)
    pages, table, _ = kv4ref.fill(rng, 2, 1, 64, 64, [700, 700])
    mass = torch.zeros((2, 1, table.shape[1] * 64), device="cuda")
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([700, 700]), ends=_ints([-(1 << 31) + 200, 3]), mass=mass)
    for q_len, dtype in ((70, torch.bfloat16), (20, torch.float32)):
        q = _dev(rng.standard_normal((2, q_len, 2, 64)), dtype)
        out, lse = cache.attend(q, accumulate=True)
        cache.check()
        assert (out[0] == 0).all() and torch.isneginf(lse[0]).all() and (out[1, :-3] == 0).all()
        assert (mass[0] == 0).all() and (mass[1, :, 3:] == 0).all() and torch.isfinite(mass).all()


def test_the_class_refuses():
    import torch
    rng = np.random.default_rng(35)
    cache = _empty_cache(2, 2, 64, 16, 4, rng, [5, 7])
    q = torch.zeros((2, 1, 4, 64), device="cuda")
    for bad in (dict(accumulate=True), dict(out=torch.zeros((2, 1, 4, 64), device="cuda", dtype=torch.float16)),
                dict(lse=torch.zeros((2, 1, 3), device="cuda")), dict(q_lens=torch.zeros(2, device="cuda"))):
        with pytest.raises(ValueError):
            cache.attend(q, **bad)
    with pytest.raises(ValueError):
        cache.attend(q[:1])
    with pytest.raises(ValueError):
        cache.attend(q.cpu())
    with pytest.raises(TypeError):
        cache.attend(q.double())
    with pytest.raises(pk.PkvError) as e:
        cache.attend(torch.zeros((2, 1, 3, 64), device="cuda"))
    assert e.value.status == L.ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError):
        cache.evict(4)
    with pytest.raises(ValueError):
        cache.append(q[:, :, :2], q[:, :, :3])
    with pytest.raises(ValueError):
        cache.read(3, torch.float16, out=(q[:, :, :2], q[:, :, :2]))
    cache.check()


# -- eviction ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim,heads,page", [(64, 2, 16), (128, 3, 64)])
@pytest.mark.parametrize("lens,budget,sinks,recent", [([100, 64, 65, 0], 64, 4, 16), ([1500, 1100], 1030, 0, 0), ([90, 128], 20, 10, 10),
                                                      ([300, 77], 1, 0, 1), ([200], 199, 3, 60)])
def test_evictions(dim, heads, page, lens, budget, sinks, recent):
    import torch
    rng = np.random.default_rng(len(lens) + budget)
    S = len(lens)
    pages, table, _ = kv4ref.fill(rng, S, heads, dim, page, [min(n, 130) for n in lens])
    max_pages = -(-max(lens) // page)
    if table.shape[1] < max_pages:  # the rows are random bytes there
        pages = rng.integers(0, 256, (S * max_pages, heads, page // 16, 18 * dim)).astype(np.uint8)
        table = rng.permutation(S * max_pages).reshape(S, max_pages).astype(np.int32)
    else:
        table = np.maximum(table, 0)
    cap = table.shape[1] * page
    ends = np.asarray(lens) + rng.integers(0, 40, S)
    pos, mass = np.full((S, heads, cap), -1, np.int32), np.zeros((S, heads, cap), np.float32)
    for s, n in enumerate(lens):
        for h in range(heads):
            pos[s, h, :n] = rng.permutation(int(ends[s]))[:n]
            mass[s, h, :n] = np.exp(3 * rng.standard_normal(n))
            mass[s, h, :n][rng.random(n) < 0.3] = rng.choice([0.0, 0.5, 0.25, np.inf, 1e-42])  # many equal
            if n > 20:
                mass[s, h, 3], mass[s, h, 11] = np.nan, -1.0
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints(lens), ends=_ints(ends), positions=_ints(pos), mass=_dev(mass))
    want_pages, want_pos, want_mass = pages.copy(), pos.copy(), mass.copy()
    for s, n in enumerate(lens):
        for h in range(heads):
            for to, fro in kv4ref.evict(pos[s, h], mass[s, h].astype(np.float64), n, int(ends[s]), budget, sinks, recent):
                for side in range(2):
                    codes, sc = kv4ref.get_row(pages[table[s, fro // page]], h, fro % page, side, dim)
                    kv4ref.put_row(want_pages[table[s, to // page]], h, to % page, side, codes, sc, dim)
                want_pos[s, h, to], want_mass[s, h, to] = pos[s, h, fro], mass[s, h, fro]
    cache.evict(budget, sinks=sinks, recent=recent)
    cache.check()
    assert np.array_equal(cache.positions.cpu().numpy(), want_pos)
    assert np.array_equal(cache.mass.cpu().numpy().view(np.uint32), want_mass.view(np.uint32))
    got = cache.pages.cpu().numpy()
    assert np.array_equal(got, want_pages), np.argwhere(got != want_pages)[:5]
    assert cache.lens.tolist() == lens


def test_eviction_of_a_sequence_longer_than_shared_memory_holds():
    import torch
    rng = np.random.default_rng(41)
    n, budget, heads, page = 60000, 20000, 1, 64
    cap = -(-n // page) * page
    pages = torch.from_numpy(rng.integers(0, 256, (cap // page, heads, page // 16, 18 * 64)).astype(np.uint8))
    table = np.arange(cap // page, dtype=np.int32)[None]
    pos, mass = np.arange(cap, dtype=np.int32).reshape(1, 1, cap), rng.random((1, 1, cap)).astype(np.float32)
    mass[..., ::7] = 0.5
    cache = kv4.Kv4Cache(pages.cuda(), _ints(table), _ints([n]), positions=_ints(pos), mass=_dev(mass))
    moves = kv4ref.evict(pos[0, 0], mass[0, 0].astype(np.float64), n, n, budget, 4, 100)
    cache.evict(budget, sinks=4, recent=100)
    cache.check()
    to, fro = np.array(moves).T
    want = pos[0, 0].copy()
    want[to] = fro
    assert np.array_equal(cache.positions.cpu().numpy()[0, 0], want)
    k = cache.read(n)[0][0, :, 0].cpu().numpy()
    cache2 = kv4.Kv4Cache(pages.cuda(), _ints(table), _ints([n]))
    k2 = cache2.read(n)[0][0, :, 0].cpu().numpy()
    assert np.array_equal(k[to].view(np.uint32), k2[fro].view(np.uint32))


# -- together --------------------------------------------------------------------------------------------------------------
def _steps(caches, steps, budget, gen, dtype, collect):
    import torch
    lens, ends = caches[0].lens, caches[0].ends
    for n in steps:
        lens += n
        ends += n
        for c in caches:
            k, v = (torch.randn((c.n_seqs, n, c.n_kv_heads, c.dim), generator=gen, device="cuda", dtype=torch.float32).to(dtype) for _ in range(2))
            q = torch.randn((c.n_seqs, n, 2 * c.n_kv_heads, c.dim), generator=gen, device="cuda", dtype=torch.float32).to(dtype)
            c.append(k, v)
            out, lse = c.attend(q, accumulate=True, window=40, sinks=2)
            c.evict(budget, sinks=2, recent=10)
            collect.append((c, k, v, q, out, lse))
        lens.clamp_(max=budget)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_append_attend_evict_over_many_steps(dtype):
    """A prompt, then tokens one by one and in drafts, two layers: at every step the attention equals that of a plain model
    of the cache (a list of (position, key, value, mass) per head)."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(1)
    S, H, d, budget = 2, 2, 64, 48
    caches = kv4.Kv4Cache.allocate(2, S, H, d, 96, page_tokens=16, evictable=True)
    log = []
    steps = [40, 1, 1, 3, 1, 8, 1, 1, 20, 1]
    _steps(caches, steps, budget, gen, _dt(dtype), log)
    for c in caches:
        c.check()
    model = {id(c): [[[] for _ in range(H)] for _ in range(S)] for c in caches}
    end, at = 0, 0
    for n in steps:
        end += n
        for c in caches:
            _, k, v, q, out, lse = log[at]
            at += 1
            kq, vq = (kv4ref.dequantise(*kv4ref.quantise(t.double().cpu().numpy())) for t in (k, v))
            q = q.double().cpu().numpy()
            for s in range(S):
                for h in range(H):
                    held = model[id(c)][s][h]
                    held += [[end - n + i, kq[s, i, h], vq[s, i, h], 0.0] for i in range(n)]
                    val = np.stack([np.stack([e[1] for e in held]), np.stack([e[2] for e in held])])[None, :, None]
                    pos = np.array([e[0] for e in held])[None, None]
                    w = kv4ref.attend(q[s:s + 1, :, 2 * h:2 * h + 2], val, [len(held)], [end], pos, 2, d ** -0.5, 40, 2, [n])
                    _close(out[s:s + 1, :, 2 * h:2 * h + 2], lse[s:s + 1, :, 2 * h:2 * h + 2], w[0], w[1], *w[3:])
                    for e, m in zip(held, w[2][0, 0]):
                        e[3] += m
                    # the gaps between weights are far above their error for these inputs, so the choice is the same
                    for to, fro in kv4ref.evict(pos[0, 0], np.array([e[3] for e in held]), len(held), end, budget, 2, 10):
                        held[to] = held[fro]
                    del held[budget:]
    for c in caches:
        pos = c.positions.cpu().numpy()
        for s in range(S):
            for h in range(H):
                assert [e[0] for e in model[id(c)][s][h]] == pos[s, h, :budget].tolist()


def test_a_decoded_pool_becomes_resident():
    """Vectors of a compressed shell, decoded to f32, go into the 4-bit cache and are attended to."""
    import torch
    from provekv_b200 import pool
    d, H, T = 64, 2, 50
    prof = pk.TurboProfile.from_seed(d, 4, 32, 42)
    x = torch.randn((T * H, d), device="cuda")
    stride = pool.payload_batch_stride(T * H, prof.record_bytes)
    payload = torch.zeros(stride, dtype=torch.uint8, device="cuda")
    err = torch.full((1,), -1, dtype=torch.int64, device="cuda")
    lay = L.Layout.make(n_tokens=T, n_heads=H, token_stride=H * d, head_stride=d)
    prof.encode_dev(x.data_ptr(), lay, payload.data_ptr(), stride, err.data_ptr())
    dec = torch.empty((1, T, H, d), device="cuda")
    prof.decode_patch_dev(payload.data_ptr(), stride, lay, dec.data_ptr(), err.data_ptr())
    pk.read_error_word(err.data_ptr())
    (cache,) = kv4.Kv4Cache.allocate(1, 1, H, d, T)
    cache.lens += T
    cache.append(dec, dec)
    k, _ = cache.read(T)
    cache.check()
    want = kv4ref.dequantise(*kv4ref.quantise(dec.double().cpu().numpy()))
    assert np.array_equal(k.double().cpu().numpy(), want)
    rel = np.linalg.norm(want - dec.double().cpu().numpy()) / np.linalg.norm(want)
    assert rel < 0.2


def test_captured_steps_replay_with_new_lengths():
    """One decode step in a CUDA graph: lengths, keys and queries change between replays, two graphs have workspaces of
    their own, and the results are those of the calls made one by one."""
    import torch
    S, H, d, G = 2, 2, 128, 2
    rng = np.random.default_rng(51)
    make = lambda: kv4.Kv4Cache.allocate(1, S, H, d, 4000, evictable=True)[0]  # noqa: E731
    live, plain = make(), make()
    pre = _dev(rng.standard_normal((S, 2100, H, d)), torch.bfloat16)
    for c in (live, plain):
        c.lens += 2100
        c.ends += 2100
        c.append(pre, pre)
    k, q = (torch.zeros((S, 1, n, d), dtype=torch.bfloat16, device="cuda") for n in (H, H * G))

    def step(c):
        c.lens += 1
        c.ends += 1
        c.append(k, k)
        return c.attend(q, accumulate=True)

    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(g, stream=side):
                outs.append(step(live))
            graphs.append(g)
    for i in range(6):
        k.copy_(_dev(rng.standard_normal((S, 1, H, d)), torch.bfloat16))
        q.copy_(_dev(rng.standard_normal((S, 1, H * G, d)), torch.bfloat16))
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        want = step(plain)
        assert torch.equal(outs[i % 2][0], want[0]) and torch.equal(outs[i % 2][1], want[1])
    assert torch.equal(live.mass, plain.mass) and torch.equal(live.pages, plain.pages) and torch.equal(live.positions, plain.positions)
    live.check()


def test_two_calls_at_once_on_two_streams():
    import torch
    rng = np.random.default_rng(52)
    pages, table, _ = kv4ref.fill(rng, 1, 1, 64, 64, [2500])
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([2500]))
    qs = [_dev(rng.standard_normal((1, 1, 4, 64)), torch.bfloat16) for _ in range(2)]
    want = [cache.attend(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        got = []
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(cache.attend(q))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_far_pages_and_sums_do_not_wrap():
    """Pages beyond 4 GiB, and a sequence in them."""
    import torch
    n_pages, page, H, d = 40000, 64, 16, 128
    pages = torch.zeros((n_pages, H, page // 16, 18 * d), dtype=torch.uint8, device="cuda")  # 5.9 GB
    assert pages.numel() > 1 << 32
    table = torch.arange(n_pages - 3, n_pages, dtype=torch.int32, device="cuda").view(1, 3)
    cache = kv4.Kv4Cache(pages, table, _ints([150]))
    x = torch.randn((1, 150, H, d), device="cuda")
    cache.append(x, x)
    k, v = cache.read(150)
    cache.check()
    want = kv4ref.dequantise(*kv4ref.quantise(x.double().cpu().numpy()))
    assert np.array_equal(k.double().cpu().numpy(), want) and torch.equal(k, v)
    assert int(pages[:n_pages - 3].max()) == 0
    q = torch.randn((1, 1, H, d), device="cuda")
    out, lse = cache.attend(q)
    w = kv4ref.attend(q.double().cpu().numpy(), np.stack([want.transpose(0, 2, 1, 3)] * 2, 1), [150], [150], None, 1, d ** -0.5, 0, 0, [1])
    _close(out, lse, w[0], w[1], *w[3:])


# -- what must not go unnoticed ------------------------------------------------------------------------------------------
def test_the_join_follows_no_entry_that_was_not_written():
    """The table of parts as a copy that never arrives leaves it: whatever lay in the workspace.  Rows of such entries are
    reported and stay as they were, the others are joined."""
    import ctypes as C
    import torch
    rng = np.random.default_rng(61)
    heads, group, n = 8, 2, 2500
    pages, table, _ = kv4ref.fill(rng, 1, heads, 64, 64, [n])
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([n]))
    q = _dev(rng.standard_normal((1, 1, heads * group, 64)), torch.float32)
    want, wlse = cache.attend(q)
    cache.check()
    lib, rows, args = L.lib(), cache._rows(q, "q"), L.Kv4AttendC(64 ** -0.5, heads * group, 0, 0, 0, 0)
    need = lib.pkv_kv4_attend_workspace_bytes(cache._ref, rows, C.byref(args))
    work = torch.zeros(need, dtype=torch.uint8, device="cuda")
    out, lse = torch.empty_like(q), torch.empty((1, 1, heads * group), device="cuda")

    def call(f):
        L.check(f(cache._ref, q.data_ptr(), rows, out.data_ptr(), rows, lse.data_ptr(), None, C.byref(args), work.data_ptr(), need,
                  cache.error.data_ptr(), torch.cuda.current_stream().cuda_stream))

    call(lib.pkv_kv4_attend_dev)
    cache.check()
    assert torch.equal(out, want) and torch.equal(lse, wlse)
    entries = work[-8 * heads:].view(torch.int32).view(heads, 2)  # (first run, runs) of each kv head
    runs = 4 * -(-heads * -(-cache.capacity // 64) // 4)
    assert (entries[:, 1] > 1).all() and int(entries.sum(1).max()) <= runs
    good = entries.clone()
    bad = torch.tensor([[-1, 3], [0, 0], [0, -5], [0, runs + 1], [runs - 1, 2], [0x7f7f7f7f, 0x7f7f7f7f]], dtype=torch.int32, device="cuda")
    for first in (0, 2):
        entries.copy_(good)
        entries[first:first + 6] = bad
        out.fill_(7.0)
        lse.fill_(7.0)
        call(lib.pkv_test_kv4_join_dev)
        with pytest.raises(pk.PkvError) as e:
            cache.check()
        assert (e.value.status, e.value.vector_index) == (L.VEC_DEVICE_WAIT, 0)
        spoilt = torch.zeros(heads * group, dtype=torch.bool, device="cuda")
        spoilt[first * group:(first + 6) * group] = True
        assert (out[0, 0, spoilt] == 7).all() and (lse[0, 0, spoilt] == 7).all()
        assert torch.equal(out[0, 0, ~spoilt], want[0, 0, ~spoilt]) and torch.equal(lse[0, 0, ~spoilt], wlse[0, 0, ~spoilt])


@pytest.mark.parametrize("dtype,q_len,group", [("bfloat16", 1, 4), ("float16", 10, 2), ("float32", 10, 3), ("bfloat16", 35, 2)])
def test_outputs_in_the_place_of_the_queries(dtype, q_len, group):
    """Weights from stored scores, from a second pass over the keys, and behind a chunk: written over q they are the same."""
    import torch
    rng = np.random.default_rng(62)
    pages, table, _ = kv4ref.fill(rng, 2, 2, 64, 16, [130, 71])
    make = lambda: kv4.Kv4Cache(_dev(pages), _ints(table), _ints([130, 71]),  # noqa: E731
                                mass=torch.zeros((2, 2, table.shape[1] * 16), device="cuda"))
    buf = _dev(rng.standard_normal((2, q_len + 1, 2 * group, 64)), _dt(dtype))
    for accumulate in (False, True):
        for at in (1, 0):  # exactly over the queries, and a token beside them
            plain, over = make(), make()
            b = buf.clone()
            q = b[:, 1:]
            want, wlse = plain.attend(q.clone(), accumulate=accumulate)
            out, lse = over.attend(q, accumulate=accumulate, out=b[:, at:at + q_len])
            plain.check()
            over.check()
            assert out.data_ptr() == b[:, at:].data_ptr()
            assert torch.equal(out, want) and torch.equal(lse, wlse) and torch.equal(over.mass, plain.mass)
            assert (over.mass != 0).any() == accumulate
            assert torch.equal(b[:, 0 if at else q_len], buf[:, 0 if at else q_len])


@pytest.mark.parametrize("dtype,q_len,group,lens", [("bfloat16", 1, 4, [50, 90]), ("float32", 1, 2, [50, 3000]), ("float32", 10, 2, [50, 90]),
                                                    ("float16", 10, 2, [50, 300]), ("bfloat16", 30, 4, [50, 300])])
def test_queries_that_are_not_finite_weigh_nothing(dtype, q_len, group, lens):
    """mass is that of the other rows, from stored scores and from a second pass over the keys; the first such row is reported."""
    import torch
    rng = np.random.default_rng(63)
    pages, table, values = kv4ref.fill(rng, 2, 2, 64, 16, lens)
    mass = torch.zeros((2, 2, table.shape[1] * 16), device="cuda")
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints(lens), mass=mass)
    q = _dev(rng.standard_normal((2, q_len, 2 * group, 64)), _dt(dtype))
    clean, _ = cache.attend(q)
    heads, last = 2 * group, q_len - 1
    rows = [(0, last, 1), (1, 0, heads - 1), (1, last, 0)]
    spoilt = torch.zeros((2, q_len, heads), dtype=torch.bool, device="cuda")
    q2 = q.clone()
    for (s, i, h), x in zip(rows, ("nan", "inf", "-inf")):
        q2[s, i, h, 7] = float(x)
        q2[s, i, h, 8] = -float(x)  # whatever the keys' signs, products of either
        spoilt[s, i, h] = True
    out, lse = cache.attend(q2, accumulate=True)
    with pytest.raises(pk.PkvError) as e:
        cache.check()
    assert (e.value.status, e.value.vector_index) == (L.VEC_NONFINITE_INPUT, (0 * q_len + last) * heads + 1)
    assert torch.isnan(out[spoilt]).all() and torch.equal(out[~spoilt], clean[~spoilt])
    ref = q.double().cpu().numpy()
    want = kv4ref.attend(ref, values, lens, lens, None, group, 0.125, 0, 0, [q_len] * 2)
    added = want[2].copy()
    for s, i, h in rows:  # less what those rows would have added
        n = lens[s] - q_len + i + 1
        added[s, h // group, :n] -= np.exp(0.125 * (values[s, 0, h // group, :n] @ ref[s, i, h]) - want[1][s, i, h])
    got = mass.double().cpu().numpy()[:, :, :added.shape[2]]
    # a weight is off by its score's error and its sum's, and rounded once a row; the difference above is of 64-bit numbers
    eps = 2.0 ** -18 * want[4].max() + 2.0 ** -22 * np.abs(want[1]).max() + 2.0 ** -19
    _within(got, added, (2 * eps + 2.0 ** -24 * q_len * group) * added + 1e-12, "mass")


def test_arguments_that_change_in_place_are_read_at_every_call():
    """A scale or a count may be a tensor of one value: nothing is kept by the tensor itself."""
    import torch
    rng = np.random.default_rng(64)
    pages, table, _ = kv4ref.fill(rng, 1, 2, 64, 16, [90])
    cap = table.shape[1] * 16
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([90]), positions=torch.arange(cap, device="cuda").int().expand(1, 2, cap).contiguous(),
                         mass=_dev(rng.random((1, 2, cap)), torch.float32))
    q = _dev(rng.standard_normal((1, 1, 4, 64)), torch.float32)
    scale, window, sinks = torch.tensor(0.125), torch.tensor(20), torch.tensor(3)
    for change in (None, (scale, -0.3), (window, 7), (sinks, 30), (window, 0)):
        if change:
            change[0].fill_(change[1])
        want = cache.attend(q, scale=float(scale), window=int(window), sinks=int(sinks))
        got = cache.attend(q, scale=scale, window=window, sinks=sinks)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(TypeError):
        cache.attend(q, window=7.0)
    budget = torch.tensor(80)
    cache.evict(budget)  # its workspace is smaller than that of the next
    cache.lens.clamp_(max=80)
    budget.fill_(40)
    cache.evict(budget)
    cache.check()


def test_more_tokens_than_32_bits_are_refused():
    """An expanded tensor has as many tokens as its view says, not those of the count's lower 32 bits."""
    import torch
    rng = np.random.default_rng(65)
    cache = _empty_cache(1, 2, 64, 16, 4, rng, [5])
    before = cache.pages.clone()
    x = torch.ones((1, 1, 2, 64), device="cuda")
    for n in ((1 << 32) + 1, 1 << 31):
        with pytest.raises(ValueError, match="tokens"):
            cache.append(x.expand(1, n, 2, 64), x.expand(1, n, 2, 64), _ints([1]))
    assert torch.equal(cache.pages, before)
    cache.append(x.expand(1, 5, 2, 64), x.expand(1, 5, 2, 64))
    cache.check()
    want = kv4ref.dequantise(*kv4ref.quantise(np.ones((1, 5, 2, 64))))  # 7 x 0.140625, the scale nearest to 1 / 7
    assert np.array_equal(cache.read(5)[0].double().cpu().numpy(), want)


def test_tensors_that_are_replaced_are_used():
    import torch
    rng = np.random.default_rng(66)
    pages, table, _ = kv4ref.fill(rng, 2, 2, 64, 16, [40, 70])
    cap = table.shape[1] * 16
    q = _dev(rng.standard_normal((2, 1, 4, 64)), torch.float32)
    make = lambda p, lens, **kw: kv4.Kv4Cache(p, _ints(table), lens, **kw)  # noqa: E731
    cache = make(_dev(pages), _ints([40, 70]))
    first = cache.attend(q)
    cache.lens += 1  # in place, then assigned to itself
    assert cache.lens.tolist() == [41, 71]
    lens = cache.lens = cache.lens - 9
    assert cache.lens is lens
    want = make(_dev(pages), _ints([32, 62])).attend(q)
    got = cache.attend(q)
    assert torch.equal(got[0], want[0]) and not torch.equal(got[0], first[0])
    more = torch.cat([_dev(pages), _dev(pages).flip(0)])  # a pool of another size
    cache.pages, cache.page_table = more, _ints(more.shape[0] - 1 - table)
    assert torch.equal(cache.attend(q)[0], want[0])
    cache.mass, cache.positions = torch.zeros((2, 2, cap), device="cuda"), torch.arange(cap, device="cuda").int().expand(2, 2, cap).contiguous()
    got = cache.attend(q, accumulate=True)
    assert torch.equal(got[0], want[0]) and (cache.mass[0, :, :32] > 0).all() and (cache.mass[0, :, 32:] == 0).all()
    cache.mass = None
    with pytest.raises(ValueError, match="mass"):
        cache.attend(q, accumulate=True)
    cache.check()
    for name, t in (("lens", _ints([1, 2, 3])), ("lens", lens.long()), ("lens", lens.cpu()), ("lens", None), ("pages", more[:, :1]),
                    ("page_table", _ints(table)[:, :1]), ("positions", torch.zeros((2, 2, 2 * cap), dtype=torch.int32, device="cuda")[:, :, ::2])):
        with pytest.raises(ValueError, match=name):
            setattr(cache, name, t)
    assert torch.equal(cache.attend(q)[0], want[0])
    with pytest.raises(AttributeError):
        cache.error = cache.error.clone()


def test_calls_are_planned_and_made_on_the_caches_device(monkeypatch):
    """As if another device were current: workspace and launch are asked for inside the guard, the device of the cache in it."""
    import torch
    rng = np.random.default_rng(67)
    pages, table, _ = kv4ref.fill(rng, 1, 1, 64, 64, [2500])
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([2500]))
    q = _dev(rng.standard_normal((1, 1, 4, 64)), torch.float32)
    events = []

    class Guard(torch.cuda.device):
        def __enter__(self):
            events.append(self.idx)
            return super().__enter__()

        def __exit__(self, *args):
            events.append("out")
            return super().__exit__(*args)

    class Recorder:
        def __getattr__(self, name):
            def call(*args):
                events.append(name)
                return getattr(L.lib(), name)(*args)
            return call

    want = cache.attend(q)
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([2500]))
    monkeypatch.setattr(torch.cuda, "device", Guard)
    cache._lib, cache._current_device = Recorder(), lambda: cache._index + 1
    got = cache.attend(q)
    assert events == [cache._index, "pkv_kv4_attend_workspace_bytes", "out", cache._index, "pkv_kv4_attend_dev", "out"]
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_refuses_to_drop_a_gradient():
    import torch
    rng = np.random.default_rng(68)
    pages, table, _ = kv4ref.fill(rng, 1, 1, 64, 16, [20])
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([20]))
    q = _dev(rng.standard_normal((1, 1, 2, 64)), torch.float32)
    want, _ = cache.attend(q)
    q.requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        cache.attend(q)
    with torch.no_grad():
        assert torch.equal(cache.attend(q)[0], want)
    assert torch.equal(cache.attend(q.detach())[0], want)


def test_read_into_slices_of_one_buffer():
    """k and v side by side in it are apart; in one place, or a head's width off, they are refused."""
    import torch
    rng = np.random.default_rng(69)
    cache = _empty_cache(2, 3, 64, 16, 3, rng, [9, 40])
    k, v = (_dev(rng.standard_normal((2, 9, 3, 64)), torch.bfloat16) for _ in range(2))
    cache.append(k, v)
    wk, wv = cache.read(9, torch.bfloat16)
    buf = torch.full((2, 9, 8, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    cache.read(9, out=(buf[:, :, 4:7], buf[:, :, :3]))
    cache.check()
    assert torch.equal(buf[:, :, 4:7], wk) and torch.equal(buf[:, :, :3], wv) and (buf[:, :, 3] == 3).all() and (buf[:, :, 7] == 3).all()
    before = buf.clone()
    for a, b in ((0, 0), (0, 2), (3, 1)):
        with pytest.raises(pk.PkvError) as e:
            cache.read(9, out=(buf[:, :, a:a + 3], buf[:, :, b:b + 3]))
        assert e.value.status == L.ERR_INVALID_ARGUMENT
    assert torch.equal(buf, before)


def test_written_vectors_that_lie_over_one_another_are_refused():
    import torch
    rng = np.random.default_rng(70)
    pages, table, _ = kv4ref.fill(rng, 2, 2, 64, 16, [30, 55])
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([30, 55]))
    q = torch.ones((2, 3, 4, 64), device="cuda")
    buf = torch.zeros(4096, device="cuda")
    for strides in ((768, 256, 0), (768, 256, 32), (768, 64, 64), (256, 256, 64), (0, 256, 64)):  # broadcast, half, sliding windows
        with pytest.raises(ValueError, match="over one another"):
            cache.attend(q, out=buf.as_strided((2, 3, 4, 64), (*strides, 1)))
    assert (buf == 0).all()
    want, _ = cache.attend(q)
    for strides in ((768, 256, 64), (64, 128, 512), (1024, 320, 68)):  # any order, gaps
        out = buf.as_strided((2, 3, 4, 64), (*strides, 1))
        cache.attend(q, out=out)
        assert torch.equal(out, want)
    one = torch.zeros(256, device="cuda").as_strided((1, 1, 4, 64), (0, 0, 64, 1))  # strides of dimensions of one say nothing
    few = kv4.Kv4Cache(_dev(pages), _ints(table[:1]), _ints([30]))
    few.attend(q[:1, :1], out=one)
    cache.check()


def test_ends_that_were_not_raised_are_reported_where_positions_are_kept():
    """lens += n alone: every call says so; with both raised none does."""
    import torch
    (cache,) = kv4.Kv4Cache.allocate(1, 3, 2, 64, 64, page_tokens=16, evictable=True)
    x = torch.ones((3, 20, 2, 64), device="cuda")
    q = torch.ones((3, 1, 4, 64), device="cuda")
    cache.lens += 20
    cache.ends += torch.tensor([20, 19, 25], dtype=torch.int32, device="cuda")
    cache.ends[2] += 5
    calls = (lambda: cache.append(x, x), lambda: cache.read(20), lambda: cache.attend(q), lambda: cache.attend(x[:, :, :1].expand(3, 20, 8, 64).bfloat16()),
             lambda: cache.evict(16))
    for call in calls:
        call()
        with pytest.raises(pk.PkvError) as e:
            cache.check()
        assert (e.value.status, e.value.vector_index) == (L.VEC_BAD_SEQUENCE, 1)
    cache.ends[1] += 1
    for call in calls:
        call()
        cache.check()


# -- the other forms, with their choice checked ---------------------------------------------------------------------------
def _launches(f):
    before = L.lib().pkv_launch_count()
    r = f()
    return r, L.lib().pkv_launch_count() - before


def _workspace(cache, q, **kw):
    import ctypes as C
    f = dict(scale=1.0, n_q_heads=q.shape[2], window=0, sinks=0, accumulate=0, max_len=0)
    f.update(kw)
    args = L.Kv4AttendC(*[f[n] for n, _ in L.Kv4AttendC._fields_])
    return L.lib().pkv_kv4_attend_workspace_bytes(cache._ref, cache._rows(q, "q"), C.byref(args))


def _splits(cache, q, **kw):
    """Of a chunk's tokens: 256 rows of partial sums each; 1 if it has no partial sums."""
    tasks = -(-q.shape[1] * q.shape[2] // cache.n_kv_heads // 256)
    return max(1, _workspace(cache, q, **kw) // (tasks * cache.n_seqs * cache.n_kv_heads * 256 * (cache.dim + 2) * 4))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("page,lens,q_len,group,window,sinks,moved", [(48, [1150], 60, 2, 0, 0, False), (16, [1300, 5, 0], 60, 1, 300, 70, True),
                                                                      (64, [1100, 1124], 25, 2, 0, 0, True), (32, [2100], 300, 1, 900, 9, False)])
def test_chunks_in_splits(dim, page, lens, q_len, group, window, sinks, moved):
    """More than 48 rows, long enough for two splits and more."""
    cache, q, _, _ = _attend_case(71 + page, "bfloat16", dim, 1, group, page, lens, q_len, window, sinks, moved, True,
                                  q_lens=[min(q_len, n + 2) for n in lens])
    assert q_len * group > 48 and _splits(cache, q, window=window, sinks=sinks) >= 2
    assert _launches(lambda: cache.attend(q, window=window, sinks=sinks))[1] == 2


def test_a_chunk_in_more_than_sixteen_splits():
    """Each row is joined by a CTA."""
    cache, q, _, _ = _attend_case(72, "float16", 64, 1, 1, 64, [9100], 50, 0, 0, False, True)
    assert _splits(cache, q) > 16
    cache, q, _, _ = _attend_case(73, "bfloat16", 128, 1, 1, 48, [9050, 100], 52, 0, 0, True, False)
    assert _splits(cache, q) > 16


@pytest.mark.parametrize("dim,dtype", [(64, "bfloat16"), (128, "float16")])
def test_a_chunk_of_many_units_in_one_cta(dim, dtype):
    """40 units and more through the rings of a CTA: enough sequences that nothing is split, a missing page far behind."""
    import torch
    rng = np.random.default_rng(74)
    S, n, q_len = 75, 2700, 50
    lens = [n] + [60] * (S - 1)
    pages, table, values = kv4ref.fill(rng, 1, 1, dim, 64, [n])
    table[0, 30] = -1
    full = np.repeat(table, S, 0)  # the others hold the first tokens of the same pages
    cache = kv4.Kv4Cache(_dev(pages), _ints(full), _ints(lens))
    q = _dev(rng.standard_normal((S, q_len, 2, dim)), _dt(dtype))
    assert _splits(cache, q) == 1
    (out, lse), launches = _launches(lambda: cache.attend(q))
    assert launches == 1
    with pytest.raises(pk.PkvError) as e:
        cache.check()
    assert (e.value.status, e.value.vector_index) == (L.VEC_BAD_SEQUENCE, 0)
    pos = np.arange(n, dtype=np.int64)[None, None].copy()
    pos[0, 0, 30 * 64:31 * 64] = 1 << 30  # beyond every query: not seen
    for s in (0, 1, S - 1):
        w = kv4ref.attend(q[s:s + 1].double().cpu().numpy(), values, [lens[s]], [lens[s]], pos, 2, dim ** -0.5, 0, 0, [q_len])
        _close(out[s:s + 1], lse[s:s + 1], w[0], w[1], *w[3:])


@pytest.mark.parametrize("page,n,q_len", [(16, 300, 60), (48, 1300, 30), (64, 1300, 70)])
def test_pages_missing_from_chunks(page, n, q_len):
    """More than 48 rows; a page missing at the start, inside and at the end of a unit, alone and across splits."""
    import torch
    rng = np.random.default_rng(75 + n)
    pages, table, values = kv4ref.fill(rng, 2, 1, 128, page, [n, 40])
    missing = [0, 2, 3, (n - 1) // page]
    for i, p in enumerate(missing):
        table[0, p] = (-1, pages.shape[0], -(1 << 31), (1 << 31) - 1)[i]
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([n, 40]), mass=torch.zeros((2, 1, table.shape[1] * page), device="cuda"))
    q = _dev(rng.standard_normal((2, q_len, 2, 128)), torch.float16)
    out, lse = cache.attend(q, accumulate=True)
    with pytest.raises(pk.PkvError) as e:
        cache.check()
    assert (e.value.status, e.value.vector_index) == (L.VEC_BAD_SEQUENCE, 0)
    pos = np.tile(np.arange(n, dtype=np.int64), (2, 1, 1))
    for p in missing:
        pos[0, 0, p * page:(p + 1) * page] = 1 << 30
    w = kv4ref.attend(q.double().cpu().numpy(), values, [n, 40], [n, 40], pos, 2, 128 ** -0.5, 0, 0, [q_len] * 2)
    _close(out, lse, w[0], w[1], *w[3:])
    mass = cache.mass[:, :, :n].double().cpu().numpy()
    assert (mass[0][pos[0] == 1 << 30] == 0).all() and (mass[0, 0, page:2 * page] > 0).all()
    eps = 2.0 ** -18 * w[4].max() + 2.0 ** -22 * np.abs(w[1][np.isfinite(w[1])]).max() + 2.0 ** -19
    _within(mass, w[2], (2 * eps + 2.0 ** -24 * q_len * 2) * w[2], "mass")


@pytest.mark.parametrize("dtype,group", [("bfloat16", 4), ("float32", 2), ("float32", 6), ("float16", 12)])
def test_a_row_for_every_warp_with_one_long_sequence(dtype, group):
    """2048 row tiles: a CTA each, nothing cut.  One sequence has more units than its warps fetch page numbers for at once."""
    import torch
    rng = np.random.default_rng(76)
    S, H, n = 256, 8, 3000
    nt = 2 if group > 8 else 1
    pages, table, values = kv4ref.fill(rng, 2, H, 64, 16, [n, 90])
    lens = rng.integers(0, 90, S)
    lens[[0, 3, S - 1]] = 0, n, 90
    full = np.repeat(table[1:], S, 0)  # short ones share a sequence's pages
    full[3] = table[0]
    cache = kv4.Kv4Cache(_dev(pages), _ints(full), _ints(lens), mass=torch.zeros((S, H, table.shape[1] * 16), device="cuda"))
    q = _dev(rng.standard_normal((S, 1, H * group, 64)), _dt(dtype))
    assert S * H * -(-group // (8 * nt)) >= 2048 and _workspace(cache, q) == 0
    (out, lse), launches = _launches(lambda: cache.attend(q))
    assert launches == 1
    again, lse2 = cache.attend(q, accumulate=True)
    cache.check()
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    for s in (0, 1, 3, 100, S - 1):
        which = 0 if s == 3 else 1
        w = kv4ref.attend(q[s:s + 1].double().cpu().numpy(), values[which:which + 1], lens[s:s + 1], lens[s:s + 1], None, group, 0.125, 0, 0, [1])
        _close(out[s:s + 1], lse[s:s + 1], w[0], w[1], *w[3:])
        if lens[s]:
            got = cache.mass[s:s + 1, :, :lens[s]].double().cpu().numpy()
            eps = 2.0 ** -18 * w[4].max() + 2.0 ** -22 * np.abs(w[1]).max() + 2.0 ** -19
            _within(got, w[2][:, :, :lens[s]], (2 * eps + 2.0 ** -24 * group) * w[2][:, :, :lens[s]], "mass")
        assert (cache.mass[s, :, lens[s]:] == 0).all()


@pytest.mark.parametrize("dtype,group", [("bfloat16", 4), ("float32", 1)])
def test_weights_whose_scores_would_not_fit(dtype, group):
    """A table of more than 256 MiB of scores: a second pass over the keys instead, with the same weights."""
    import torch
    rng = np.random.default_rng(77)
    n, page = 2000, 64
    pages, table, values = kv4ref.fill(rng, 1, 2, 64, page, [n])
    small = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([n]), mass=torch.zeros((1, 2, table.shape[1] * page), device="cuda"))
    slots = (1 << 22) + 64  # x 2 heads x 8 rows x 4 bytes
    wide = np.full((1, slots // page), -1, np.int32)
    wide[:, :table.shape[1]] = table
    large = kv4.Kv4Cache(_dev(pages), _ints(wide), _ints([n]), mass=torch.zeros((1, 2, slots), device="cuda"))
    q = _dev(rng.standard_normal((1, 1, 2 * group, 64)), _dt(dtype))
    assert _workspace(large, q, accumulate=1) == _workspace(large, q) and _workspace(small, q, accumulate=1) > _workspace(small, q)
    a, b = small.attend(q, accumulate=True), large.attend(q, accumulate=True)
    small.check()
    large.check()
    w = kv4ref.attend(q.double().cpu().numpy(), values, [n], [n], None, group, 0.125, 0, 0, [1])
    eps = 2.0 ** -18 * w[4].max() + 2.0 ** -22 * np.abs(w[1]).max() + 2.0 ** -19
    for cache, (out, lse) in ((small, a), (large, b)):
        _close(out, lse, w[0], w[1], *w[3:])
        _within(cache.mass[:, :, :n].double().cpu().numpy(), w[2][:, :, :n], (2 * eps + 2.0 ** -24 * group) * w[2][:, :, :n], "mass")
    assert (large.mass[:, :, n:] == 0).all()


@pytest.mark.parametrize("dim,heads,cap,n,budget", [(128, 2, 9984, 9984, 4000), (64, 1, 16384, 16000, 15900), (128, 1, 49152, 30011, 200),
                                                    (128, 1, 49216, 20000, 19000), (64, 2, 131072, 2112, 2048)])
def test_evictions_from_long_tables(dim, heads, cap, n, budget):
    """More than 8192 slots: 1024 threads, keys in shared memory up to 49152 slots and read again beyond; short lists are moved
    by the same launch, long ones by a second."""
    import torch
    rng = np.random.default_rng(cap + n)
    page = 64
    pages = rng.integers(0, 256, (cap // page, heads, page // 16, 18 * dim)).astype(np.uint8)
    table = rng.permutation(cap // page).reshape(1, -1).astype(np.int32)
    end = n + 100
    pos, mass = np.full((1, heads, cap), -1, np.int32), np.zeros((1, heads, cap), np.float32)
    for h in range(heads):
        pos[0, h, :n] = rng.permutation(end)[:n]
        mass[0, h, :n] = np.where(rng.random(n) < 0.4, 0.5, np.exp(3 * rng.standard_normal(n)))  # the budget cuts equal weights
    cache = kv4.Kv4Cache(_dev(pages), _ints(table), _ints([n]), ends=_ints([end]), positions=_ints(pos), mass=_dev(mass))
    _, launches = _launches(lambda: cache.evict(budget, sinks=4, recent=budget // 4))
    cache.check()
    assert launches == (1 if min(cap - budget, budget) <= 256 else 2)
    want_pos, want_mass, rows = pos.copy(), mass.copy(), pages[table[0]].copy()  # slot order
    for h in range(heads):
        moves = kv4ref.evict(pos[0, h], mass[0, h].astype(np.float64), n, end, budget, 4, budget // 4)
        assert moves
        for to, fro in moves:
            for side in range(2):
                codes, sc = kv4ref.get_row(pages[table[0, fro // page]], h, fro % page, side, dim)
                kv4ref.put_row(rows[to // page], h, to % page, side, codes, sc, dim)
            want_pos[0, h, to], want_mass[0, h, to] = pos[0, h, fro], mass[0, h, fro]
    assert np.array_equal(cache.positions.cpu().numpy(), want_pos)
    assert np.array_equal(cache.mass.cpu().numpy(), want_mass)
    assert np.array_equal(cache.pages[cache.page_table[0].long()].cpu().numpy(), rows)
