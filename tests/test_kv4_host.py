"""The 4-bit KV cache without a GPU: refusals of the C calls (made before anything is launched), the checks of the
Python class, and the plain restatement the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import kv4ref
from provekv_b200 import _lib as L
from provekv_b200 import kv4

P = 1 << 20  # a pointer that is only looked at for its alignment


def _cache(**kw):
    f = dict(pages=P, page_table=P, lens=P, ends=None, positions=None, mass=None, n_pages=8, dim=128, n_kv_heads=2,
             page_tokens=64, n_seqs=2, max_pages=4, reserved=0)
    f.update(kw)
    return L.Kv4CacheC(*[f[n] for n, _ in L.Kv4CacheC._fields_])


def _rows(n=1, dtype=L.DST_BF16, strides=(1024, 512, 128)):
    return L.Kv4RowsC(*strides, n, dtype)


def _append(cache, k=P, kr=None, v=P, vr=None, err=P, fn="pkv_kv4_append_dev"):
    kr, vr = kr or _rows(), vr or _rows()
    rest = (0,) if fn == "pkv_kv4_read_dev" else ()
    return getattr(L.lib(), fn)(C.byref(cache), k, C.byref(kr), v, C.byref(vr), None, *rest, err, None)


@pytest.mark.parametrize("fn", ["pkv_kv4_append_dev", "pkv_kv4_read_dev"])
def test_append_and_read_refuse(fn):
    bad, unsup = L.ERR_INVALID_ARGUMENT, L.ERR_UNSUPPORTED
    for kw, want in ((dict(pages=None), bad), (dict(pages=P + 8), bad), (dict(lens=None), bad), (dict(positions=P + 4), bad), (dict(mass=P + 8), bad), (dict(page_table=None), bad),
                     (dict(reserved=1), bad), (dict(n_kv_heads=0), bad), (dict(n_seqs=-1), bad), (dict(max_pages=-1), bad),
                     (dict(page_tokens=0), bad), (dict(n_pages=-1), bad), (dict(dim=96), unsup), (dict(dim=256), unsup),
                     (dict(page_tokens=24), unsup), (dict(max_pages=1 << 26), unsup), (dict(n_seqs=70000), unsup)):
        assert _append(_cache(**kw), fn=fn) == want, kw
    c = _cache()
    assert _append(c, k=None, fn=fn) == bad and _append(c, v=P + 4, fn=fn) == bad and _append(c, err=None, fn=fn) == bad
    assert _append(c, kr=_rows(dtype=3), fn=fn) == bad
    assert _append(c, kr=_rows(dtype=L.DST_F16), fn=fn) == bad                      # k and v of different types
    assert _append(c, kr=_rows(2), fn=fn) == bad                                    # or lengths
    assert _append(c, kr=_rows(strides=(1024, 516, 128)), fn=fn) == bad             # 16-bit rows off 16-byte boundaries
    f32 = lambda s: _rows(dtype=L.DST_F32, strides=s)  # noqa: E731
    assert _append(c, kr=f32((1024, 514, 128)), vr=f32((1024, 512, 128)), fn=fn) == bad
    many = _rows(4 * 64 + 1)
    assert _append(c, kr=many, vr=many, fn=fn) == bad                               # more tokens than a sequence has slots
    none = _rows(0)
    assert _append(c, k=None, v=None, kr=none, vr=none, fn=fn) == L.OK              # nothing to do
    assert _append(_cache(n_seqs=0), fn=fn) == L.OK


def _attend(cache, args, q=P, qr=None, out=P, outr=None, lse=P, work=None, bytes_=0, err=P):
    qr, outr = qr or _rows(), outr or _rows()
    return L.lib().pkv_kv4_attend_dev(C.byref(cache), q, C.byref(qr), out, C.byref(outr), lse, None, C.byref(args), work, bytes_,
                                      err, None)


def _args(**kw):
    f = dict(scale=1.0, n_q_heads=4, window=0, sinks=0, accumulate=0, max_len=0)
    f.update(kw)
    return L.Kv4AttendC(*[f[n] for n, _ in L.Kv4AttendC._fields_])


def test_attend_refuses():
    bad = L.ERR_INVALID_ARGUMENT
    c = _cache()
    for kw in (dict(n_q_heads=3), dict(n_q_heads=0), dict(window=-1), dict(sinks=-1), dict(max_len=-1), dict(accumulate=2),
               dict(scale=float("nan")), dict(scale=float("inf")), dict(accumulate=1)):
        assert _attend(c, _args(**kw)) == bad, kw
    assert _attend(_cache(mass=P), _args(accumulate=1), lse=None) == bad
    assert _attend(c, _args(), q=None) == bad and _attend(c, _args(), out=P + 2) == bad and _attend(c, _args(), err=None) == bad
    assert _attend(c, _args(), outr=_rows(2)) == bad and _attend(c, _args(), outr=_rows(dtype=L.DST_F32)) == bad
    assert _attend(_cache(dim=80), _args()) == L.ERR_UNSUPPORTED
    assert _attend(c, _args(), qr=_rows(0), outr=_rows(0)) == L.OK
    # a long cache is split over CTAs: the partial sums need room
    long = _cache(max_pages=4096, n_seqs=1)
    qr = _rows()
    need = L.lib().pkv_kv4_attend_workspace_bytes(C.byref(long), C.byref(qr), C.byref(_args()))
    assert need > 0 and need % 8 == 0
    assert _attend(long, _args(), work=P, bytes_=need - 1) == L.ERR_BUFFER_TOO_SMALL
    assert _attend(long, _args(), work=P + 8, bytes_=need) == bad
    assert L.lib().pkv_kv4_attend_workspace_bytes(C.byref(long), C.byref(qr), C.byref(_args(n_q_heads=3))) == 0
    assert L.lib().pkv_kv4_attend_workspace_bytes(C.byref(long), C.byref(qr), C.byref(_args(max_len=100))) == 0


def test_evict_refuses():
    bad, f = L.ERR_INVALID_ARGUMENT, L.lib().pkv_kv4_evict_dev
    full = _cache(positions=P, mass=P)
    call = lambda c, b, s, r, w=P, n=1 << 30, e=P: f(C.byref(c), b, s, r, w, n, e, None)  # noqa: E731
    assert call(_cache(mass=P), 64, 0, 0) == bad and call(_cache(positions=P), 64, 0, 0) == bad
    assert call(full, 0, 0, 0) == bad and call(full, 64, -1, 0) == bad and call(full, 64, 0, -1) == bad
    assert call(full, 64, 60, 5) == bad and call(full, 64, 0, 0, e=None) == bad
    assert call(full, 64, 0, 0, n=8) == L.ERR_BUFFER_TOO_SMALL and call(full, 64, 0, 0, w=None) == bad
    assert call(full, 256, 0, 0, w=None, n=0) == L.OK  # the budget is the capacity: nothing can be over it
    assert L.lib().pkv_kv4_evict_workspace_bytes(C.byref(full), 64) == 2 * 2 * (2 * 64 + 1) * 4


def test_status_of_a_bad_sequence_has_a_text():
    assert "sequence" in L.status_string(L.VEC_BAD_SEQUENCE)


def test_the_class_checks_its_tensors():
    import torch
    pages = torch.zeros((4, 2, 4, 18 * 128), dtype=torch.uint8)
    table, lens = torch.zeros((1, 4), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kv4.Kv4Cache(pages, table, lens)
    with pytest.raises(ValueError, match="18"):
        kv4.Kv4Cache(pages[..., :18 * 96], table, lens)
    with pytest.raises(ValueError, match="lens"):
        kv4.Kv4Cache(pages, table, lens.long())
    with pytest.raises(ValueError, match="lens"):
        kv4.Kv4Cache(pages, table, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="mass"):
        kv4.Kv4Cache(pages, table, lens, mass=torch.zeros((1, 2, 255)))
    with pytest.raises(ValueError, match="contiguous"):
        kv4.Kv4Cache(pages.transpose(0, 2), table, lens)


# -- the restatement itself ------------------------------------------------------------------------------------------
def test_scales_are_the_upper_bits_of_binary16():
    bits = (np.arange(0xDF).astype(np.uint16) << 7).view(np.float16).astype(np.float64)
    assert np.array_equal(bits, kv4ref.SCALES)


def test_scale_rounding_against_a_search():
    rng = np.random.default_rng(0)
    amax = np.concatenate([np.exp(rng.uniform(-13, 10.7, 4000)), 7 * kv4ref.SCALES, 3.5 * (kv4ref.SCALES[1:] + kv4ref.SCALES[:-1]), [0.0]])
    got = kv4ref.scale_codes(amax)
    for a, c in zip(amax, got):
        dist = np.abs(kv4ref.SCALES - a / 7)
        best = np.flatnonzero(dist == dist.min())
        assert c == (best[best % 2 == 0][0] if len(best) > 1 else best[0])
    assert kv4ref.scale_codes(7 * 7424.0) == 0xDE and kv4ref.scale_codes(7 * 7424.5) == -1


def test_values_are_exact_in_both_16_bit_types_and_near_the_input():
    import torch
    rng = np.random.default_rng(1)
    x = rng.standard_normal((50, 128)) * np.exp(rng.uniform(-8, 7, (50, 1)))
    y = kv4ref.dequantise(*kv4ref.quantise(x))
    for t in (torch.float16, torch.bfloat16):
        assert np.array_equal(torch.from_numpy(y).to(t).double().numpy(), y)
    # half a step, and the scale is within 1/17 of amax / 7 (8 of 3 + 1 bits: half a unit in 8.5)
    amax = np.abs(x.reshape(50, -1, 16)).max(-1, keepdims=True)
    step = amax / 7 * (1 + 1 / 17)
    assert (np.abs(x - y).reshape(50, -1, 16) <= 0.5 * step * (1 + 1e-12)).all()


def test_rows_come_back_from_a_page():
    rng = np.random.default_rng(2)
    for dim in (64, 128):
        page = rng.integers(0, 256, (2, 3, 18 * dim)).astype(np.uint8)
        want = {}
        for h in range(2):
            for t in range(48):
                for side in range(2):
                    want[h, t, side] = (rng.integers(0, 16, dim).astype(np.uint8), rng.integers(0, 0xDF, dim // 16).astype(np.uint8))
                    kv4ref.put_row(page, h, t, side, *want[h, t, side], dim)
        for (h, t, side), (c, s) in want.items():
            gc, gs = kv4ref.get_row(page, h, t, side, dim)
            assert np.array_equal(c, gc) and np.array_equal(s, gs)


def test_allocate_refuses_pages_of_no_whole_atoms():
    for page in (0, 8, 40, -16):
        with pytest.raises(ValueError, match="multiple of 16"):
            kv4.Kv4Cache.allocate(1, 1, 1, 64, 100, page_tokens=page, device="cpu")


def test_counts_do_not_wrap():
    assert kv4._int32("window", (1 << 31) - 1) == (1 << 31) - 1
    for x in (-1, 1 << 31, (1 << 32) + 5):
        with pytest.raises(ValueError, match="window"):
            kv4._int32("window", x)


def test_the_join_alone_is_there_for_split_rows_only():
    f = L.lib().pkv_test_kv4_join_dev
    row = _rows(dtype=L.DST_F32)
    call = lambda c, n: f(C.byref(c), P, C.byref(row), P, C.byref(row), P, None, C.byref(_args()), P, n, P, None)  # noqa: E731
    assert call(_cache(dim=64), 1 << 30) == L.ERR_UNSUPPORTED                                # short rows: nothing is cut
    assert call(_cache(dim=128, max_pages=4096, n_seqs=1), 1 << 30) == L.ERR_UNSUPPORTED
    assert call(_cache(dim=64, max_pages=4096, n_seqs=1), 8) == L.ERR_BUFFER_TOO_SMALL


def test_attend_refuses_outputs_over_its_queries():
    """By the vectors, not by the ranges: q, k and v of one buffer lie between one another without meeting."""
    bad = L.ERR_INVALID_ARGUMENT
    full = _cache(mass=P, max_pages=4096, n_seqs=2)           # needs a workspace: where nothing is refused the call ends there
    rows = lambda s: _rows(3, strides=s)  # noqa: E731
    packed = (3 * 12 * 128, 12 * 128, 128)                     # 12 heads side by side, 4 of them queries
    for shift, strides, acc, want in ((0, packed, 0, None), (0, packed, 1, bad), (4 * 128 * 2, packed, 1, None), (3 * 128 * 2, packed, 0, bad),
                                      (-8 * 128 * 2, packed, 1, None), (-9 * 128 * 2, packed, 1, bad), (12 * 128 * 2, packed, 0, bad),
                                      (3 * 12 * 128 * 2, packed, 0, bad), (6 * 12 * 128 * 2, packed, 1, None),
                                      (16, packed, 0, bad), (-16, packed, 0, bad), (4 * 128 * 2 - 16, packed, 0, bad),
                                      (0, (3 * 512, 512, 128), 0, bad), (6 * 12 * 128 * 2, (3 * 512, 512, 128), 1, None),
                                      (-6 * 512 * 2, (3 * 512, 512, 128), 1, None), (-6 * 512 * 2 + 16, (3 * 512, 512, 128), 0, bad)):
        got = _attend(full, _args(accumulate=acc), q=P, out=P + shift, qr=rows(packed), outr=rows(strides))
        assert got == (want or L.ERR_BUFFER_TOO_SMALL), (shift, strides, acc)


def test_overlap_against_a_list_of_bytes():
    rng = np.random.default_rng(3)
    full = _cache(dim=64, max_pages=4096, n_seqs=3, n_kv_heads=1)
    seen = set()
    for _ in range(400):
        counts = (3, int(rng.integers(1, 5)), int(rng.integers(1, 4)))
        order, step, strides = rng.permutation(3), 64, [0, 0, 0]
        for i in order:  # axes in any order with gaps of whole vectors between them
            strides[i] = int(step + 64 * rng.integers(0, 3))
            step = strides[i] * counts[i]
        shift = int(rng.integers(-step // 8 - 8, step // 8 + 8)) * 8 * 2
        at = np.add.outer(np.add.outer(np.arange(counts[0]) * strides[0], np.arange(counts[1]) * strides[1]), np.arange(counts[2]) * strides[2])
        q = (at.reshape(-1, 1) + np.arange(64)).ravel()
        want = shift != 0 and np.isin(q, q + shift // 2).any()
        row = _rows(counts[1], strides=tuple(strides))
        got = _attend(full, _args(n_q_heads=counts[2]), q=P, out=P + shift, qr=row, outr=row)
        assert (got == L.ERR_INVALID_ARGUMENT) == want and got in (L.ERR_INVALID_ARGUMENT, L.ERR_BUFFER_TOO_SMALL), (counts, strides, shift)
        seen.add(bool(want))
    assert seen == {False, True}


def test_counts_become_plain_numbers():
    import torch
    for x in (np.int64(7), torch.tensor(7), True):
        assert type(kv4._int32("sinks", x)) is int and kv4._int32("sinks", x) == int(x)
    for x in (1.0, torch.tensor(1.5), "3"):
        with pytest.raises(TypeError):
            kv4._int32("sinks", x)


def test_rows_share_runs_only_where_their_units_can_be_numbered():
    """2^24 units of 64 tokens in the table, 1024 row tiles: 2^34 units, whatever bound on the lengths the caller gives."""
    need = lambda c, **kw: L.lib().pkv_kv4_attend_workspace_bytes(C.byref(c), C.byref(_rows()), C.byref(_args(n_q_heads=16, **kw)))  # noqa: E731
    huge = dict(max_pages=1 << 24, n_seqs=64, n_kv_heads=16)
    assert need(_cache(**huge)) == 0
    assert need(_cache(**huge), max_len=1 << 17) == 0
    assert need(_cache(**huge), window=1 << 17) > 0                    # a window bounds what is visited
    assert need(_cache(**huge, positions=P), window=1 << 17) == 0      # unless any slot may be in it
    assert need(_cache(**{**huge, "max_pages": 1 << 20}), max_len=1 << 17) > 0


@pytest.mark.parametrize("fn", ["pkv_kv4_append_dev", "pkv_kv4_read_dev"])
def test_token_numbers_stay_in_32_bits(fn):
    """Rows up to the last tile's end are numbered; n_seqs = 0 would end the call before anything is launched."""
    f = getattr(L.lib(), fn)
    rest = (0,) if fn == "pkv_kv4_read_dev" else ()
    for n, want in ((0x7fff0000, L.OK), (0x7fff0001, L.ERR_UNSUPPORTED), (0x7fffffff, L.ERR_UNSUPPORTED)):
        row = _rows(n, strides=(0, 0, 128))
        assert f(C.byref(_cache(n_seqs=0)), P, C.byref(row), P, C.byref(row), P, *rest, P, None) == want


def test_read_refuses_outputs_over_one_another():
    packed = (2 * 5 * 6 * 128, 6 * 128, 128)  # k and v heads side by side, three sequences
    call = lambda shift: L.lib().pkv_kv4_read_dev(C.byref(_cache(n_kv_heads=3)), P, C.byref(_rows(5, strides=packed)), P + shift,  # noqa: E731
                                                  C.byref(_rows(5, strides=packed)), None, 0, P, None)
    for shift in (0, 128 * 2, -2 * 128 * 2, 16, 6 * 128 * 2):
        assert call(shift) == L.ERR_INVALID_ARGUMENT, shift
