"""History cache without a GPU: the oracle's rules against hand-worked values, and every refusal of the entry points
(the C ABI checks its arguments on the host before it touches the device)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import hist as oh
from tests import hist_cases


def test_oracle_8_bit_rows_by_hand():
    # 448 is the largest code: a row with maximum 448 keeps exponent 0, one step more moves to exponent 1
    v, e = oh.quantise(np.array([[448.0, 1.0, 17.0, 0.0], [448.5, 1.0, -17.0, 18.0]]))
    assert e.tolist() == [0, 1]
    assert v[0].tolist() == [448.0, 1.0, 16.0, 0.0]             # 17 lies between 16 and 18: the even one
    assert v[1].tolist() == [448.0, 1.0, -16.0, 18.0]           # 448.5 / 2 -> 224; 8.5 is a tie -> 8; 9 is a code
    # maximum just above a power of two: exponent floor(log2) - 8
    v, e = oh.quantise(np.array([[1.0, 2.0 ** -14, 2.0 ** -18, 0.0]]))
    assert e.tolist() == [-8] and v[0].tolist() == [1.0, 2.0 ** -14, 0.0, 0.0]   # 2^-18 * 2^8 = half of 2^-9: to 0
    # infinities and NaN do not set the exponent and come back as NaN
    v, e = oh.quantise(np.array([[np.inf, 2.0, -np.inf, np.nan]]))
    assert e.tolist() == [-7] and np.isnan(v[0]).tolist() == [True, False, True, True] and v[0, 1] == 2.0
    v, e = oh.quantise(np.zeros((1, 4)))
    assert e.tolist() == [-126] and not v.any()
    # every e4m3 value is its own rounding (torch's codes as the independent table)
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    codes = codes[np.isfinite(codes)]
    assert np.array_equal(oh.e4m3_round(codes), codes) and codes.max() == oh.E4M3_MAX


def test_oracle_rounding_equals_torchs_cast():
    rng = np.random.default_rng(3)
    x = (rng.standard_normal(200000) * np.exp2(rng.uniform(-12, 6, 200000))).astype(np.float32)
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(oh.e4m3_round(x), want)


def test_oracle_places():
    table = np.array([[4, 0, -1], [2, 9, 1]])
    # 5 pages of 16: sequence 0 owns rows 0..2 as its positions 15, 16, 17; sequence 1 row 3 as position 40, in page 1
    where, bad = oh.places(5, [0, 3, 4], 2, table, 16, 5, [18, 41])
    assert where == [(4, 15), (0, 0), (0, 1), (1, 8), 'none'] and not bad
    where, bad = oh.places(4, None, 2, table, 16, 5, [1, 20])    # position -1: no place; positions 18, 19 on page 9: bad
    assert where == [None, (4, 0), None, None] and bad


def test_oracle_attention_of_one_position_is_its_value():
    rng = np.random.default_rng(0)
    kv = rng.standard_normal((3, 2, 2, 16, 32))
    q = rng.standard_normal((2, 1, 4, 32))
    out, _, _ = oh.attention(kv, q, np.array([[2], [0]]), [1, 0], 0.1, 16)
    for h in range(4):
        np.testing.assert_allclose(out[0, 0, h], kv[2, h // 2, 1, 0], rtol=0, atol=0)
    assert not out[1].any()


# ------------------------------------------------------------------------------------------------ refusals (C ABI)
def _cache(**over):
    from recommendation_amd import _lib
    args = dict(kv=4096, exps=None, n_pages=8, n_heads=2, page_size=16, dim=64, dtype=_lib.MI_DT_BF16)
    args.update(over)
    return _lib.HistCacheC(**args)


@pytest.mark.parametrize('over, text', [
    (dict(kv=None), 'null cache'), (dict(kv=4104), 'aligned'), (dict(dtype=3), 'dtype'), (dict(dim=48), 'dim'), (dict(dim=16), 'dim'),
    (dict(dim=512), 'dim'), (dict(page_size=8), 'page_size'), (dict(page_size=48), 'page_size'),
    (dict(page_size=2048), 'page_size'), (dict(n_heads=0), 'n_heads'), (dict(n_pages=0), 'n_pages'),
    (dict(n_pages=1 << 31), 'n_pages'), (dict(exps=4096), 'exps'), (dict(dtype=2), 'exps'),
])
def test_bad_caches_are_refused(over, text):
    from recommendation_amd import _lib
    lib = _lib.load()
    c = _cache(**over)
    calls = [
        lambda: lib.mi_hist_write(ctypes.byref(c), 4096, 4096, 1, 128, 64, 128, 64, 4, None, 4, 4096, 2, 2, 4096, None, None),
        lambda: lib.mi_hist_read(ctypes.byref(c), 4096, 4096, 1, 128, 64, 128, 64, 4, None, 4, 4096, 2, 2, 4096, None, None),
        lambda: lib.mi_hist_attn(ctypes.byref(c), 4096, 128, 128, 64, 2, 1, 4, 4096, 2, 2, 4096, 0.1, 4096, 128, 128, 64, None,
                                 0, None, None)]
    for call in calls:
        assert call() == -1 and text in lib.mi_last_error().decode(), lib.mi_last_error()


def test_bad_row_calls_are_refused():
    from recommendation_amd import _lib
    lib = _lib.load()
    c = _cache()

    def rc(k=4096, v=4096, dtype=1, strides=(128, 64, 128, 64), n=4, offsets=None, seqs=4, table=4096, ld=2, width=2,
           lengths=4096):
        out = {lib.mi_hist_write(ctypes.byref(c), k, v, dtype, *strides, n, offsets, seqs, table, ld, width, lengths, None, None),
               lib.mi_hist_read(ctypes.byref(c), k, v, dtype, *strides, n, offsets, seqs, table, ld, width, lengths, None, None)}
        assert len(out) == 1
        return out.pop(), lib.mi_last_error().decode()

    for kw, text in [(dict(k=None), 'null rows'), (dict(v=None), 'null rows'), (dict(dtype=2), 'f32 or bf16'),
                     (dict(k=4104), '16-byte'), (dict(strides=(128, 64, 132, 64)), '16-byte'),
                     (dict(strides=(128, 4, 128, 64)), '16-byte'), (dict(n=-1), 'n_rows'), (dict(n=6), 'divide'),
                     (dict(table=None), 'page table'), (dict(lengths=None), 'lengths'), (dict(width=0), 'width'),
                     (dict(ld=1), 'width'), (dict(seqs=-1), 'n_seqs')]:
        code, msg = rc(**kw)
        assert code == -1 and text in msg, (kw, msg)
    code, msg = rc(n=1 << 30, offsets=4096)                      # 2^32 rows of K and V
    assert code == -4 and 'in one call' in msg
    assert rc(n=0)[0] == 0 and rc(seqs=0)[0] == 0                # nothing to do: no launch, no error


def test_bad_attention_calls_are_refused():
    from recommendation_amd import _lib
    lib = _lib.load()
    c = _cache()

    def rc(q=4096, qs=(128, 128, 64), heads=2, tokens=1, seqs=4, table=4096, ld=2, width=2, lengths=4096, out=4096,
           os_=(128, 128, 64)):
        code = lib.mi_hist_attn(ctypes.byref(c), q, *qs, heads, tokens, seqs, table, ld, width, lengths, 0.1, out, *os_, None, 0,
                                None, None)
        return code, lib.mi_last_error().decode()

    for kw, text in [(dict(q=None), 'null q'), (dict(out=None), 'null q or out'), (dict(heads=3), '3 heads'),
                     (dict(heads=0), '0 heads'), (dict(tokens=-1), 'queries'), (dict(qs=(128, 128, 60)), '16-byte'),
                     (dict(out=4100), '16-byte'), (dict(table=None), 'page table'), (dict(width=0), 'width'),
                     (dict(lengths=None), 'lengths'), (dict(tokens=70000), 'query rows')]:
        code, msg = rc(**kw)
        assert code == -1 and text in msg, (kw, msg)
    assert rc(tokens=0)[0] == 0 and rc(seqs=0)[0] == 0


def test_attention_workspace_is_checked():
    """Page tables of up to 1024 positions need none; beyond, what mi_hist_attn_workspace_bytes says."""
    from recommendation_amd import _lib
    lib = _lib.load()
    c = _cache()
    need = lambda **kw: lib.mi_hist_attn_workspace_bytes(ctypes.byref(_cache(**kw.pop('cache', {}))), kw.pop('seqs', 4), kw.pop('tokens', 1),
                                                         kw.pop('heads', 2), kw.pop('width', 65))
    assert need(width=16) == need(width=64) == 0 and need() > 0
    assert need(seqs=0) == need(tokens=0) == need(heads=3) == need(width=0) == need(cache=dict(dim=48)) == 0
    assert need(seqs=4096, width=4096) < 1 << 26

    def rc(ws, ws_bytes, width=65, seqs=4, ld=100000000, tokens=1):
        code = lib.mi_hist_attn(ctypes.byref(c), 4096, 128, 128, 64, 2, tokens, seqs, 4096, ld, width, 4096, 0.1, 4096, 128, 128,
                                64, ws, ws_bytes, None, None)
        return code, lib.mi_last_error().decode()

    for ws, n in ((None, 0), (None, 1 << 30), (4096, need() - 1), (4096, 0)):
        code, msg = rc(ws, n)
        assert code == -3 and 'workspace' in msg and str(need()) in msg, (ws, n, msg)
    code, msg = rc(4104, 1 << 30)
    assert code == -1 and 'aligned' in msg
    # more work than one launch can number
    for kw in (dict(seqs=1 << 26), dict(width=100000000, seqs=1 << 10), dict(seqs=1 << 14, tokens=65536)):
        code, msg = rc(4096, 1 << 40, **kw)
        assert code == -4 and 'in one call' in msg, (kw, code, msg)


def test_host_tensors_are_refused():
    from recommendation_amd import ops
    with pytest.raises(ops.MiError, match='device tensors'):
        ops.HistCache(4, 16, 2, 64, device='cpu')
    for bad in (dict(page_size=8), dict(page_size=24), dict(dim=48), dict(n_pages=0)):
        args = dict(n_pages=4, page_size=16, n_heads=2, dim=64)
        args.update(bad)
        with pytest.raises(ops.MiError, match='HistCache'):
            ops.HistCache(device='cpu', **args)
    with pytest.raises(TypeError, match='HistCache'):
        ops.HistCache(4, 16, 2, 64, dtype=torch.float16, device='cpu')


def test_results_that_overlap_are_refused():
    """An expanded result (a stride of zero, or below a row's length) would take several rows in one place, in no order.
    Inputs may be expanded, and the stride of a dimension of one entry says nothing."""
    from recommendation_amd import _lib
    lib = _lib.load()
    one = _cache(n_heads=1)

    def read(strides, c=None, n=4, offsets=4096):
        code = lib.mi_hist_read(ctypes.byref(c or _cache()), 4096, 4096, 1, *strides, n, offsets, 4, 4096, 2, 2, 4096, None, None)
        return code, lib.mi_last_error().decode()

    for strides in ((0, 64, 128, 64), (128, 64, 0, 64), (128, 0, 128, 64), (128, 64, 128, 0), (56, 64, 128, 64), (-128, 64, 128, 64)):
        code, msg = read(strides)
        assert code == -1 and 'overlap' in msg, (strides, msg)
    # one row, one head: those strides are not looked at; the call goes on to the next check (rows of one call)
    for strides, c in (((128, 0, 128, 0), one), ((64, 0, 64, 0), one)):
        code, msg = read(strides, c, n=1 << 30)
        assert code == -4 and 'in one call' in msg, (strides, code, msg)

    def attn(os_, tokens=2, seqs=4, heads=2, width=65):
        code = lib.mi_hist_attn(ctypes.byref(_cache()), 4096, 0, 0, 0, heads, tokens, seqs, 4096, width, width, 4096, 0.1, 4096,
                                *os_, None, 0, None, None)
        return code, lib.mi_last_error().decode()

    for os_ in ((0, 128, 64), (256, 0, 64), (256, 128, 0), (256, 128, 32)):
        code, msg = attn(os_)
        assert code == -1 and 'overlap' in msg, (os_, msg)
    for os_, kw in (((256, 128, 64), {}), ((128, 0, 64), dict(tokens=1)), ((0, 128, 64), dict(seqs=1))):
        code, msg = attn(os_, **kw)                               # past that check: the workspace is the next
        assert code == -3 and 'workspace' in msg, (os_, kw, msg)


def test_results_whose_rows_meet_are_refused():
    """Rows that share memory across two dimensions, K and V rows in one place, and a result that is partly its own
    queries: each stride by itself looks right."""
    from recommendation_amd import _lib
    lib = _lib.load()
    base = 1 << 20

    def read(k, v, strides, n=4, offsets=4096):
        code = lib.mi_hist_read(ctypes.byref(_cache(n_heads=3)), k, v, 1, *strides, n, offsets, 4, 4096, 2, 2, 4096, None, None)
        return code, lib.mi_last_error().decode()

    far = base << 4
    for k, v, strides in [
            (base, base, (192, 64, 192, 64)),                       # the same tensor twice
            (base, far, (64, 64, 192, 64)), (far, base, (192, 64, 64, 64)),   # row stride = head stride (unfolded)
            (base, far, (128, 64, 192, 64)), (base, far, (64, 128, 192, 64)),
            (base, base + 2 * 64, (192, 64, 192, 64)),              # V's heads are K's next heads
            (base, base + 2 * 192, (192, 64, 192, 64)),             # V's rows are K's next rows
            (base, base + 2 * 3 * 192, (192, 64, 192, 64)),         # ... the last one only
            (base + 2 * 3 * 192, base, (192, 64, 192, 64)),
            (base, base + 16, (384, 64, 384, 64)),                  # half a row apart
            (base, base, (192, 64, 64, 256))]:                      # the same memory, heads in front in V
        code, msg = read(k, v, strides)
        assert code == -1 and 'overlap' in msg, (k, v, strides, code, msg)

    def attn(q, qs, out, os_, tokens=2, seqs=4, heads=2, width=2):
        code = lib.mi_hist_attn(ctypes.byref(_cache()), q, *qs, heads, tokens, seqs, 4096, width, width, 4096, 0.1, out, *os_, None,
                                0, None, None)
        return code, lib.mi_last_error().decode()

    plain = (256, 128, 64)
    for q, qs, out, os_ in [
            (far, plain, base, (256, 64, 64)), (far, plain, base, (64, 256, 64)), (far, plain, base, (128, 128, 64)),
            (far, plain, base, (128, 64, 128)),
            (base, plain, base, (256, 64, 128)),                    # tokens and heads exchanged
            (base, plain, base + 2 * 64, plain), (base, plain, base + 2 * 256, plain), (base + 2 * 3 * 256, plain, base, plain),
            (base, (512, 128, 64), base, plain), (base, (0, 128, 64), base, plain), (base, plain, base + 16, plain)]:
        code, msg = attn(q, qs, out, os_)
        assert code == -1 and 'overlap' in msg, (q, qs, out, os_, code, msg)
    # past every check on the rows of out, the workspace is the next: transposed results, results with gaps
    for os_ in ((256, 64, 128), (64, 512, 256), (512, 128, 64), (72, 576, 288)):
        code, msg = attn(far, plain, base, os_, width=65)
        assert code == -3 and 'workspace' in msg, (os_, code, msg)


def test_one_table_row_for_all_sequences():
    """Row stride 0 (an expanded table): taken where the pages are only read, refused where they are written."""
    from recommendation_amd import _lib
    lib = _lib.load()

    def attn(ld):
        code = lib.mi_hist_attn(ctypes.byref(_cache()), 1 << 20, 128, 128, 64, 2, 1, 4, 4096, ld, 65, 4096, 0.1, 1 << 21, 128, 128, 64,
                                None, 0, None, None)
        return code, lib.mi_last_error().decode()

    code, msg = attn(0)                                              # the workspace is the next check
    assert code == -3 and 'workspace' in msg
    for ld in (-65, -1, 1, 64):
        code, msg = attn(ld)
        assert code == -1 and 'row stride' in msg, (ld, code, msg)
    args = (1 << 20, 1 << 21, 1, 128, 64, 128, 64)
    # more rows than one call can number: the check behind the table's
    assert lib.mi_hist_read(ctypes.byref(_cache()), *args, 1 << 30, 4096, 4, 4096, 0, 2, 4096, None, None) == -4
    assert lib.mi_hist_write(ctypes.byref(_cache()), *args, 1 << 30, 4096, 4, 4096, 0, 2, 4096, None, None) == -1
    assert 'row stride' in lib.mi_last_error().decode()


@pytest.mark.parametrize('dtype', [0, 1, 2])
@pytest.mark.parametrize('case', hist_cases.CUTS)
def test_the_long_cases_take_the_cuts_they_are_for(dtype, case):
    """More units than workgroups, whole rows or runs that cross them: a change of the rules must not leave them untested."""
    users, shortest, longest, heads, group, tokens, dim, aligned, run = case
    lens = hist_cases.lengths_for(np.random.default_rng(users), users, shortest, longest)
    cut = hist_cases.cut_of(dtype, lens, -(-longest // 16), 16, heads, group, tokens, dim)
    assert cut['aligned'] == aligned and cut['run'] >= run, cut
    seen = {(c['RT'], c['NR'], c['NG'] > 1, c['aligned']) for c in (
        hist_cases.cut_of(dtype, hist_cases.lengths_for(np.random.default_rng(x[0]), *x[:3]), -(-x[2] // 16), 16, *x[3:7])
        for x in hist_cases.CUTS)}
    assert {(1, 1, False, True), (2, 2, False, True), (2, 4, True, True), (1, 2, False, True), (1, 1, False, False),
            (2, 2, False, False), (2, 4, True, False), (1, 4, False, False)} <= seen


def test_counting_histories_show_a_lost_tile():
    """Planted in the sums: without any one position, tile of 16 or unit of 128, some channel is off by more than the bound that
    the attention is held to (2^-8 of the sum in 16 bits)."""
    rows, sums = hist_cases.counting_rows(np.random.default_rng(2), 3000, 2, 32)
    assert np.array_equal(np.cumsum(rows, 0), sums[1:]) and np.abs(sums[:, :, 1:]).max() <= 24
    bound = np.abs(sums[3000]) * 2.0 ** -8 + 2.0 ** -20
    for size in (1, 16, 128):
        for at in range(0, 3000, size):
            lost = sums[min(at + size, 3000)] - sums[at]
            assert (np.abs(lost) > bound)[:, 1:].any(1).all(), (size, at)
