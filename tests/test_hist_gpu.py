"""History cache on the GPU: hist_write / hist_read bit for bit and hist_attn within derived bounds of oracle/hist.py.

Bounds of the attention, per output element, with P|v| = sum_j p_j |v_jd| and u = 2^-24 (half an f32 step):
  scores     a dot product of `dim` exact or f32 products accumulated in f32, scaled twice: off by at most
             (dim + 4) u A, A = max_j sum_d |q_d k_jd| * scale; the weights exp(s_j - m) then by
             ds = 2 (dim + 4) u A + 8 u (max subtracted, exponential), numerator and denominator: 2 ds P|v|
  sums       n terms in f32, numerator and denominator: 2 (n + 16) u P|v|
  8, 16 bit  weights rounded to bf16, delta <= 2^-8 each, divided by the sum of the ROUNDED weights:
             o' - o = sum p delta (v - o) / sum p (1 + delta), at most 2^-8 (1 + 2^-7) (P|v| + |o|);
             the output rounded to bf16: 2^-8 of itself
"""
import numpy as np
import pytest
import torch

from oracle import hist as oh
from tests import hist_cases
from tests.errlog import held

pytestmark = pytest.mark.gpu

DTYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'e4m3': torch.float8_e4m3fn}
U = 2.0 ** -24


def bound(cache, dim, n, want, absv, size):
    ds = 2 * (dim + 4) * U * size[..., None] + 8 * U
    b = (2 * ds + 2 * (n + 16) * U) * absv
    if cache != 'f32':
        b = b + 2.0 ** -8 * (1 + 2.0 ** -7) * (absv + np.abs(want))
        b = b + 2.0 ** -8 * (np.abs(want) + b)
    return b + 1e-37


def poisoned(dev, cache, n_pages, page, heads, dim):
    """A cache whose every byte is a NaN."""
    from recommendation_amd import ops
    c = ops.HistCache(n_pages, page, heads, dim, dtype=DTYPES[cache], device=dev)
    if cache == 'e4m3':
        c.kv.view(torch.uint8).fill_(0x7f)
        c.exps.fill_(255)
    else:
        c.kv.fill_(float('nan'))
    return c


def values(c):
    """The cache as the float64 values it stands for."""
    if c.exps is None:
        return c.kv.double().cpu().numpy()
    return np.ldexp(c.kv.cpu().double().numpy(), c.exps.cpu().numpy().astype(np.int64)[..., None] - 127)


def tables(rng, lens, page, width, n_pages):
    """A shuffled page table with -1 behind every history; distinct pages."""
    t = np.full((len(lens), width), -1, np.int32)
    order = rng.permutation(n_pages)
    at = 0
    for b, n in enumerate(lens):
        k = -(-max(n, 0) // page)
        t[b, :k] = order[at:at + k]
        at += k
    assert at <= n_pages
    return t


def filled(dev, rng, cache, lens, page, heads, dim, spare=3, given=torch.float32, width=None, scale_rows=True):
    """A cache with random histories written through hist_write; everything else in it is NaN."""
    from recommendation_amd import ops
    need = sum(-(-max(n, 0) // page) for n in lens)
    width = width or max(1, max(-(-max(n, 0) // page) for n in lens)) + 1
    c = poisoned(dev, cache, need + spare, page, heads, dim)
    t = tables(rng, lens, page, width, need + spare)
    own = [max(n, 0) for n in lens]
    offs = np.concatenate([[0], np.cumsum(own)]).astype(np.int64)
    k = rng.standard_normal((int(offs[-1]), heads, dim))
    v = rng.standard_normal((int(offs[-1]), heads, dim))
    if scale_rows:
        v *= np.exp2(rng.integers(-3, 4, size=(int(offs[-1]), heads, 1)))
    table, lengths = torch.from_numpy(t).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    if offs[-1]:
        ops.hist_write(c, torch.from_numpy(k).to(dev, given), torch.from_numpy(v).to(dev, given), table, lengths,
                       offsets=torch.from_numpy(offs).to(dev))
    return c, table, lengths, t


# ------------------------------------------------------------------------------------------------ write and read
@pytest.mark.parametrize('given', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
@pytest.mark.parametrize('dim, heads, page', [(32, 1, 16), (64, 3, 16), (128, 2, 64), (256, 5, 32)])
def test_write_and_read_are_exact(dev, cache, given, dim, heads, page):
    from recommendation_amd import ops
    rng = np.random.default_rng(dim + heads)
    lens = [0, 1, 15, 16, 17, 40, 3, 100, 33, 5]
    new = [0, 1, 15, 7, 17, 0, 3, 64, 1, 2]
    width = 8
    n_pages = 40
    t = tables(rng, lens, page, width, n_pages)
    offs = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
    n = int(offs[-1]) + 4                                                    # four rows behind the last sequence
    x = rng.standard_normal((n, 2, heads, dim)) * np.exp2(rng.integers(-30, 30, size=(n, 2, heads, 1)))
    x[3] = 0.0
    x[4, :, 0, 0], x[5, 1, 0, 1] = np.inf, -np.inf
    x[6, 0, heads - 1, 2] = np.nan
    x[7] *= 1e-38 / np.abs(x[7]).max()                                       # exponents at the bottom
    rows = torch.from_numpy(x).to(dev, given)
    k, v = rows[:, 0], rows[:, 1]                                            # strided: K and V side by side
    c = poisoned(dev, cache, n_pages, page, heads, dim)
    want = values(c)
    err = ops.new_error_word(dev)
    table, lengths, offsets = torch.from_numpy(t).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), \
        torch.from_numpy(offs).to(dev)
    ops.hist_write(c, k, v, table, lengths, offsets=offsets, err=err)
    where, bad = oh.places(n, offs, len(lens), t, page, n_pages, lens)
    assert not bad and err.item() == 0
    held_rows = rows.double().cpu().numpy()
    if cache == 'e4m3':
        held_rows, exponents = oh.quantise(held_rows)
        for i, w in enumerate(where):
            if isinstance(w, tuple):
                got = c.exps[w[0], :, :, w[1]].cpu().numpy().astype(np.int64) - 127
                assert np.array_equal(got, exponents[i].T)
    elif cache == 'bf16':
        held_rows = torch.from_numpy(held_rows).to(torch.bfloat16).double().numpy()
    oh.write(want, held_rows[:, 0], held_rows[:, 1], where)
    np.testing.assert_array_equal(values(c), want)                           # every other byte is still a NaN
    for dtype in (torch.float32, torch.bfloat16):
        out = tuple(torch.full((n, heads, dim), 7.0, dtype=dtype, device=dev) for _ in range(2))
        ops.hist_read(c, table, lengths, offsets=offsets, out=out, err=err)
        wk, wv = np.full((n, heads, dim), 7.0), np.full((n, heads, dim), 7.0)
        oh.read(want, where, wk, wv)
        for got, w in ((out[0], wk), (out[1], wv)):
            w = torch.from_numpy(w).to(torch.float32).to(dtype)
            np.testing.assert_array_equal(got.float().cpu().numpy(), w.float().numpy())
    assert err.item() == 0


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
def test_rows_of_any_stride_and_table_views(dev, cache):
    """Heads in front of tokens, K and V of one fused projection, outputs with gaps, a page table inside a wider one; the same
    calls captured into a graph."""
    from recommendation_amd import ops
    rng = np.random.default_rng(23)
    page, heads, dim, lens = 16, 3, 64, [40, 9, 100]
    n = sum(lens)
    dt = torch.float32 if cache == 'f32' else torch.bfloat16
    t = tables(rng, lens, page, 7, 20)
    wide = torch.full((3, 16), -1, dtype=torch.int32, device=dev)
    wide[:, 5:12] = torch.from_numpy(t).to(dev)
    table, lengths = wide[:, 5:12], torch.tensor(lens, dtype=torch.int32, device=dev)
    offs = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64, device=dev)
    fused = torch.from_numpy(rng.standard_normal((n, 9 * dim + 32))).to(dev, dt)
    k = fused[:, 32:32 + heads * dim].view(n, heads, dim)
    v = torch.from_numpy(rng.standard_normal((heads, n, dim))).to(dev, dt).transpose(0, 1)
    plain, c = poisoned(dev, cache, 20, page, heads, dim), poisoned(dev, cache, 20, page, heads, dim)
    ops.hist_write(plain, k.contiguous(), v.contiguous(), table.contiguous(), lengths, offsets=offs)
    out = torch.full((n, 2, heads, dim + 16), 5.0, dtype=dt, device=dev)
    pair = (out[:, 0, :, :dim], out[:, 1, :, 16:])
    ops.hist_read(plain, table, lengths, offsets=offs, out=pair)             # also outside capture: nothing is set up
    first = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.hist_write(c, k, v, table, lengths, offsets=offs)
        ops.hist_read(c, table, lengths, offsets=offs, out=pair)
    for _ in range(3):
        c.kv.view(torch.uint8).fill_(0x7f)
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(values(c)[t[t >= 0]], np.where(np.isnan(values(plain)[t[t >= 0]]),
                                                                     values(c)[t[t >= 0]], values(plain)[t[t >= 0]]))
        assert torch.equal(out, first)
    k1, v1 = ops.hist_read(plain, table, lengths, n, offsets=offs, dtype=dt)
    assert torch.equal(pair[0], k1) and torch.equal(pair[1], v1)
    assert bool((out[:, 0, :, dim:] == 5.0).all()) and bool((out[:, 1, :, :16] == 5.0).all())


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
def test_captured_strided_writes_touch_their_rows_alone(dev, cache):
    """Byte for byte over the whole pool: pages of no table, slots behind a history and in front of the appended rows keep
    what they held, eager and in every replay, with rows of any stride and rows nobody owns among them."""
    from recommendation_amd import ops
    rng = np.random.default_rng(29)
    page, heads, dim, n_pages, lens, new = 16, 3, 64, 20, [40, 9, 0, 100], [17, 9, 2, 33]
    dt = torch.float32 if cache == 'f32' else torch.bfloat16
    n = sum(new) + 3                                                         # three rows behind the last sequence
    t = tables(rng, lens, page, 7, n_pages)
    wide = torch.full((4, 16), 11, dtype=torch.int32, device=dev)
    wide[:, 5:12] = torch.from_numpy(t).to(dev)
    table, lengths = wide[:, 5:12], torch.tensor(lens, dtype=torch.int32, device=dev)
    offs = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
    offsets = torch.from_numpy(offs).to(dev)
    fused = torch.zeros((n, heads * dim + 64), dtype=dt, device=dev)
    k, v = fused[:, 32:32 + heads * dim].view(n, heads, dim), torch.zeros((heads, n, dim), dtype=dt, device=dev).transpose(0, 1)
    c = poisoned(dev, cache, n_pages, page, heads, dim)
    where, bad = oh.places(n, offs, len(lens), t, page, n_pages, lens)
    assert not bad and 'none' in where and None in where
    touched = torch.zeros((n_pages, heads, 2, page), dtype=torch.bool)
    for w in where:
        if isinstance(w, tuple):
            touched[w[0], :, :, w[1]] = True
    touched = touched.to(dev)

    def clear():
        c.kv.view(torch.uint8).fill_(0xff)                                   # NaN in every type
        if cache == 'e4m3':
            c.exps.fill_(255)

    def check(rows):
        kept = c.kv.view(torch.uint8).view(n_pages, heads, 2, page, -1)[~touched]
        assert bool((kept == 0xff).all()) and (cache != 'e4m3' or bool((c.exps[~touched] == 255).all()))
        want = rows if cache == 'f32' else torch.from_numpy(rows).to(torch.bfloat16).double().numpy()
        if cache == 'e4m3':
            want = oh.quantise(want)[0]
        full = values(c)
        for i, w in enumerate(where):
            if isinstance(w, tuple):
                np.testing.assert_array_equal(full[w[0], :, :, w[1]], want[i].transpose(1, 0, 2))

    def draw():
        rows = rng.standard_normal((n, 2, heads, dim)).astype(np.float32).astype(np.float64)
        k.copy_(torch.from_numpy(rows[:, 0]))
        v.copy_(torch.from_numpy(rows[:, 1]))
        clear()
        return rows

    rows = draw()
    ops.hist_write(c, k, v, table, lengths, offsets=offsets)
    check(rows)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.hist_write(c, k, v, table, lengths, offsets=offsets)
    for _ in range(3):
        rows = draw()
        g.replay()
        check(rows)


def test_every_code_and_exponent_byte_of_an_8_bit_cache(dev):
    """A pool that the caller filled: each of the 256 codes under bytes from 0 (a row of zeros) to 254, in 64 bits rounded once."""
    from recommendation_amd import ops
    page, dim = 16, 256
    c = poisoned(dev, 'e4m3', 1, page, 1, dim)
    codes = torch.arange(256, dtype=torch.uint8, device=dev)
    c.kv.view(torch.uint8)[:] = codes
    each = torch.tensor([0, 1, 2, 3, 60, 100, 118, 126, 127, 128, 140, 200, 246, 247, 253, 254], dtype=torch.uint8, device=dev)
    c.exps[:] = each
    table, lengths = torch.zeros((1, 1), dtype=torch.int32, device=dev), torch.tensor([16], dtype=torch.int32, device=dev)
    want = codes.view(torch.float8_e4m3fn).double()[None] * torch.exp2(each.double() - 127)[:, None]
    want[0] = torch.where(torch.isnan(want[0]), want[0], 0.0)
    for dtype in (torch.float32, torch.bfloat16):
        k, v = ops.hist_read(c, table, lengths, 16, dtype=dtype)
        w = want.to(torch.float32).to(dtype)                                 # the f32 product is exact or infinite
        for x in (k, v):
            np.testing.assert_array_equal(x[:, 0].float().cpu().numpy(), w.float().cpu().numpy())


def test_rows_without_a_place(dev):
    """Lengths shorter than the rows given, padded sequences, bad pages and histories beyond the table."""
    from recommendation_amd import ops
    rng = np.random.default_rng(1)
    page, heads, dim, n_pages = 16, 2, 64, 10
    lens = [2, 0, 20, 36, -5, 40]
    t = np.array([[3, -1], [0, 0], [7, 10], [1, 2], [4, 4], [5, -3]], np.int32)
    offs = np.array([0, 4, 6, 12, 18, 20, 30], np.int64)
    x = rng.standard_normal((30, 2, heads, dim))
    rows = torch.from_numpy(x).to(dev, torch.bfloat16)
    table, lengths = torch.from_numpy(t).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    where, bad = oh.places(30, offs, 6, t, page, n_pages, lens)
    assert bad and None in where
    for cache in ('bf16', 'e4m3'):
        c, err = poisoned(dev, cache, n_pages, page, heads, dim), ops.new_error_word(dev)
        want = values(c)
        held_rows = rows.double().cpu().numpy()
        if cache == 'e4m3':
            held_rows = oh.quantise(held_rows)[0]
        oh.write(want, held_rows[:, 0], held_rows[:, 1], where)
        ops.hist_write(c, rows[:, 0], rows[:, 1], table, lengths, offsets=torch.from_numpy(offs).to(dev), err=err)
        np.testing.assert_array_equal(values(c), want)
        with pytest.raises(ops.InvalidArgumentError, match='out of bounds'):
            ops.check_error_word(err, 'pages')
        k, v = ops.hist_read(c, table, lengths, 30, offsets=torch.from_numpy(offs).to(dev), dtype=torch.float32, err=err)
        wk, wv = np.zeros((30, heads, dim)), np.zeros((30, heads, dim))
        oh.read(want, where, wk, wv)
        np.testing.assert_array_equal(k.cpu().numpy(), wk.astype(np.float32))
        np.testing.assert_array_equal(v.cpu().numpy(), wv.astype(np.float32))
        assert err.item() == 1
    # without an error word the same call just skips
    ops.hist_write(c, rows[:, 0], rows[:, 1], table, lengths, offsets=torch.from_numpy(offs).to(dev))
    # padded sequences alone are no error
    err = ops.new_error_word(dev)
    ops.hist_write(c, rows[:2, 0], rows[:2, 1], table[1:3], torch.tensor([0, 1], dtype=torch.int32, device=dev), err=err)
    assert err.item() == 0


@pytest.mark.parametrize('users', [1, 63, 64, 65, 700, 5000])
def test_offsets_of_many_sequences(dev, users):
    """Every search depth: empty sequences, runs of them at both ends, and one event each without offsets."""
    from recommendation_amd import ops
    rng = np.random.default_rng(users)
    page, heads, dim = 16, 1, 32
    new = rng.integers(0, 4, size=users)
    new[:users // 3] = 0
    new[-(users // 5):] = 0
    if users == 1:
        new[:] = 3
    lens = (new + rng.integers(0, 10, size=users)).astype(np.int32)
    t = tables(rng, lens, page, 1, users + 2)
    offs = np.concatenate([[0], np.cumsum(new)]).astype(np.int64)
    n = int(offs[-1])
    x = torch.from_numpy(rng.standard_normal((n, 2, heads, dim))).to(dev, torch.float32)
    c = poisoned(dev, 'f32', users + 2, page, heads, dim)
    want = values(c)
    table, lengths = torch.from_numpy(t).to(dev), torch.from_numpy(lens).to(dev)
    ops.hist_write(c, x[:, 0], x[:, 1], table, lengths, offsets=torch.from_numpy(offs).to(dev))
    where, bad = oh.places(n, offs, users, t, page, users + 2, lens)
    assert not bad
    oh.write(want, x[:, 0].double().cpu().numpy(), x[:, 1].double().cpu().numpy(), where)
    np.testing.assert_array_equal(values(c), want)
    one = torch.from_numpy(rng.standard_normal((users, 2, heads, dim))).to(dev, torch.float32)
    lengths = (lengths + 1).to(torch.int32).clamp(max=16)
    live = t[:, 0] >= 0
    ops.hist_write(c, one[:, 0], one[:, 1], table, lengths)
    k, v = ops.hist_read(c, table, lengths, users, dtype=torch.float32)
    np.testing.assert_array_equal(k.cpu().numpy()[live], one[:, 0].cpu().numpy()[live])
    np.testing.assert_array_equal(v.cpu().numpy()[live], one[:, 1].cpu().numpy()[live])
    assert not k.cpu().numpy()[~live].any()


# ------------------------------------------------------------------------------------------------ attention
def run_attn(dev, rng, cache, lens, page, heads, group, tokens, dim, width=None, name='', scale=None, queries=None):
    from recommendation_amd import ops
    c, table, lengths, t = filled(dev, rng, cache, lens, page, heads, dim, width=width)
    dt = torch.float32 if cache == 'f32' else torch.bfloat16
    n, Hq = len(lens), heads * group
    q = rng.standard_normal((n, tokens, Hq, dim)) * 1.5 if queries is None else queries
    q = torch.from_numpy(q).to(dev, dt)
    out = torch.full((n, tokens, Hq, dim + 16), 3.0, dtype=dt, device=dev)   # rows with a gap behind them
    err = ops.new_error_word(dev)
    got = ops.hist_attn(c, q, table, lengths, scale=scale, out=out[..., :dim], err=err)
    assert got.data_ptr() == out.data_ptr() and err.item() == 0
    assert bool((out[..., dim:] == 3.0).all())
    s = dim ** -0.5 if scale is None else scale
    want, absv, size = oh.attention(values(c), q.double().cpu().numpy(), t, lens, s, page)
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    b = bound(cache, dim, max(max(lens), 1), want, absv, size)
    held("hist_attn %s dim %d page %d heads %dx%d tokens %d %s" % (cache, dim, page, heads, group, tokens, name),
         (np.abs(got - want) / b).max(), 1.0)
    for i, x in enumerate(lens):
        if x <= 0:
            assert not got[i].any()
    return c, table, lengths, q, out


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 48, 63, 64, 65, 100, 127, 128, 129, 200, 0]


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
@pytest.mark.parametrize('dim', [32, 64, 128, 256])
@pytest.mark.parametrize('room', [256, 1024, 2048])
def test_attention_at_every_edge_of_tile_and_page(dev, cache, dim, room):
    """A wave, a workgroup and a run of the cut to each history: chosen by what the page table has room for."""
    rng = np.random.default_rng(dim)
    for page, heads, group, tokens in ((16, 1, 1, 1), (64, 2, 4, 1), (32, 3, 5, 2), (128, 1, 7, 5)):
        run_attn(dev, rng, cache, EDGES, page, heads, group, tokens, dim, width=room // page, name='room %d' % room)


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
@pytest.mark.parametrize('lens, heads, group, tokens, dim, page', [
    ([5000], 1, 1, 1, 64, 16), ([1023, 1, 0, 4097], 2, 8, 1, 128, 64), ([3000, 10, 2999], 1, 16, 1, 64, 1024),
    ([2500, 700], 2, 3, 11, 32, 32), ([1500, 1], 1, 1, 70, 256, 16), ([900] * 40, 4, 2, 1, 64, 16),
    ([700, 31, 400], 1, 1, 150, 64, 16), ([300, 290], 2, 1, 40, 128, 32), ([40000, 5], 1, 2, 1, 32, 256)])
def test_attention_over_long_histories(dev, cache, lens, heads, group, tokens, dim, page):
    run_attn(dev, np.random.default_rng(len(lens) + dim), cache, lens, page, heads, group, tokens, dim)


def one_history(dev, rng, cache, k, v, page):
    """A cache that holds one history of rows k, v, everything else NaN; its page table of one row."""
    from recommendation_amd import ops
    n, heads, dim = k.shape
    width = -(-n // page)
    c = poisoned(dev, cache, width + 3, page, heads, dim)
    table = torch.from_numpy(tables(rng, [n], page, width, width + 3)).to(dev)
    ops.hist_write(c, torch.from_numpy(k).to(dev, torch.float32), torch.from_numpy(v).to(dev, torch.float32), table,
                   torch.tensor([n], dtype=torch.int32, device=dev))
    return c, table


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
@pytest.mark.parametrize('case', hist_cases.CUTS, ids=lambda x: '-'.join(str(y) for y in x[:7]))
def test_every_position_counts_once_however_the_work_is_cut(dev, cache, case):
    """Equal keys: all weights are 1 and all sums whole numbers, exact in f32 in any order, so an element times the length is
    off by the division (8 u) and in 16 bits by the result's rounding (2^-8) of the sum, and by nothing where that is 0."""
    from recommendation_amd import ops
    users, shortest, longest, heads, group, tokens, dim = case[:7]
    rng = np.random.default_rng(users)
    lens = hist_cases.lengths_for(rng, users, shortest, longest)
    rows, sums = hist_cases.counting_rows(rng, longest, heads, dim)
    k = np.broadcast_to(rng.standard_normal((1, heads, dim)), rows.shape)
    c, table = one_history(dev, rng, cache, np.ascontiguousarray(k), rows, 16)
    q = torch.from_numpy(rng.standard_normal((users, tokens, heads * group, dim))).to(dev, torch.float32 if cache == 'f32' else torch.bfloat16)
    out = ops.hist_attn(c, q, table.expand(users, -1), torch.tensor(lens, dtype=torch.int32, device=dev))
    n = np.maximum(np.array(lens), 0)
    want = np.repeat(sums[n], group, 1)[:, None]                              # [users, 1, q heads, dim]
    got = out.double().cpu().numpy() * n[:, None, None, None]
    assert (np.abs(got - want) <= np.abs(want) * (8 * U + (0 if cache == 'f32' else 2.0 ** -8))).all()


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
@pytest.mark.parametrize('case', hist_cases.CUTS, ids=lambda x: '-'.join(str(y) for y in x[:7]))
def test_attention_however_the_work_is_cut(dev, cache, case):
    """Random rows, each history held to its own bound, with the additions that really follow each other in its sums."""
    from recommendation_amd import ops
    users, shortest, longest, heads, group, tokens, dim = case[:7]
    rng = np.random.default_rng(users)
    lens = hist_cases.lengths_for(rng, users, shortest, longest)
    k, v = rng.standard_normal((2, longest, heads, dim))
    c, table = one_history(dev, rng, cache, k, v * np.exp2(rng.integers(-3, 4, size=(longest, heads, 1))), 16)
    q = torch.from_numpy(rng.standard_normal((users, tokens, heads * group, dim)) * 1.5).to(dev, torch.float32 if cache == 'f32' else torch.bfloat16)
    out = ops.hist_attn(c, q, table.expand(users, -1), torch.tensor(lens, dtype=torch.int32, device=dev)).double().cpu().numpy()
    t = np.broadcast_to(table.cpu().numpy(), (users, table.shape[1]))
    cut = hist_cases.cut_of(ops.HistCache._DTYPES[DTYPES[cache]], lens, t.shape[1], 16, heads, group, tokens, dim)
    held_values, q = values(c), q.double().cpu().numpy()
    worst = 0.0
    for b in range(users):
        want, absv, size = oh.attention(held_values, q[b:b + 1], t[b:b + 1], lens[b:b + 1], dim ** -0.5, 16)
        limit = bound(cache, dim, hist_cases.depth_of(cut, max(lens[b], 0)), want, absv, size)
        worst = max(worst, (np.abs(out[b:b + 1] - want) / limit).max())
    held("hist_attn %s cut %s run %d" % (cache, '-'.join(str(y) for y in case[:7]), cut['run']), worst, 1.0)


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
def test_attention_of_many_short_histories(dev, cache):
    """The DIN shape: thousands of samples with up to 100 events, one head."""
    rng = np.random.default_rng(9)
    lens = rng.integers(0, 101, size=1500).tolist()
    run_attn(dev, rng, cache, lens, 16, 1, 1, 1, 64, width=7)


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
def test_attention_of_many_uneven_histories(dev, cache):
    """More sequences than a workgroup has threads, lengths below zero, runs of empty ones, histories that end anywhere
    in a run of the cut."""
    rng = np.random.default_rng(10)
    lens = rng.integers(0, 600, size=700)
    lens[100:160] = 0
    lens[200:400] = rng.integers(-3, 3, size=200)
    lens[0] = 1
    run_attn(dev, rng, cache, lens.tolist(), 16, 1, 2, 1, 32)
    lens[-1] = 3001
    run_attn(dev, rng, cache, lens.tolist(), 16, 1, 2, 1, 32)


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
@pytest.mark.parametrize('dim', [32, 64, 128, 256])
def test_pools_beyond_the_last_level_cache(dev, cache, dim):
    """A pool of more than 256 MB is read past the caches; same sums, bit for bit, as over the same pages in a small one."""
    rng = np.random.default_rng(dim + 1)
    page, heads = 64, 2
    for lens in ([100, 0, 1, 150], [700, 0, 1, 90], [700, 0, 1, 1500]):
        pool_beyond(dev, rng, cache, dim, page, heads, lens)


def pool_beyond(dev, rng, cache, dim, page, heads, lens):
    from recommendation_amd import ops
    c, table, lengths, t = filled(dev, rng, cache, lens, page, heads, dim)
    per_page = heads * 2 * page * dim * c.kv.element_size()
    n_pages = (300 << 20) // per_page + c.n_pages
    big = poisoned(dev, cache, n_pages, page, heads, dim)
    lo = n_pages - c.n_pages
    big.kv.view(torch.uint8)[lo:] = c.kv.view(torch.uint8)
    if cache == 'e4m3':
        big.exps[lo:] = c.exps
    moved = torch.where(table >= 0, table + lo, table)
    dt = torch.float32 if cache == 'f32' else torch.bfloat16
    for shape in ((4, 6, dim), (4, 9, 4, dim)):
        q = torch.from_numpy(rng.standard_normal(shape)).to(dev, dt)
        assert torch.equal(ops.hist_attn(big, q, moved, lengths), ops.hist_attn(c, q, table, lengths))


@pytest.mark.parametrize('cache, given', [('f32', torch.float32), ('bf16', torch.bfloat16), ('e4m3', torch.float32),
                                          ('e4m3', torch.bfloat16)])
def test_rows_beyond_the_last_level_cache(dev, cache, given):
    """A call that moves more than 256 MB goes past the caches; same bits as two calls of half the rows."""
    from recommendation_amd import ops
    gen = torch.Generator(device=dev).manual_seed(3)
    heads, dim, page, users, each = 8, 256, 256, 8, 5001
    width = -(-each // page)
    rows = torch.randn((users * each, 2, heads, dim), generator=gen, device=dev).to(given)
    assert rows.numel() * (rows.element_size() + DTYPES[cache].itemsize) > 256 << 20
    table = torch.randperm(users * width, generator=gen, device=dev).to(torch.int32).view(users, width)
    lengths = torch.full((users,), each, dtype=torch.int32, device=dev)
    whole, halves = (poisoned(dev, cache, users * width, page, heads, dim) for _ in range(2))
    ops.hist_write(whole, rows[:, 0], rows[:, 1], table, lengths)
    h = users // 8
    for b in range(0, users, h):
        part = rows[b * each:(b + h) * each]
        ops.hist_write(halves, part[:, 0], part[:, 1], table[b:b + h], lengths[b:b + h])
    assert torch.equal(whole.kv.view(torch.uint8), halves.kv.view(torch.uint8))
    if cache == 'e4m3':
        assert torch.equal(whole.exps, halves.exps)
    k, v = ops.hist_read(whole, table, lengths, users * each, dtype=given)
    for b in range(0, users, h):
        k1, v1 = ops.hist_read(whole, table[b:b + h], lengths[b:b + h], h * each, dtype=given)
        assert torch.equal(k[b * each:(b + h) * each], k1) and torch.equal(v[b * each:(b + h) * each], v1)
    if cache != 'e4m3':
        assert torch.equal(k, rows[:, 0]) and torch.equal(v, rows[:, 1])


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
def test_attention_with_peaked_and_flat_scores(dev, cache):
    """One position takes all the weight, early or late; and scale 0: the plain mean."""
    rng = np.random.default_rng(4)
    lens = [300, 77, 1]
    run_attn(dev, rng, cache, lens, 16, 2, 2, 1, 64, scale=4.0, name='peaked')
    run_attn(dev, rng, cache, lens, 16, 2, 2, 1, 64, scale=0.0, name='mean')
    run_attn(dev, rng, cache, lens, 16, 2, 2, 1, 64, scale=-0.3, name='negative scale')


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
@pytest.mark.parametrize('power', [None, -100, -60, 60, 90])
def test_attention_over_rows_of_zeros_and_of_extreme_size(dev, cache, power):
    """Value rows of zeros (their weights count all the same), and keys and values of very small or large size."""
    from recommendation_amd import ops
    rng = np.random.default_rng(17)
    for lens in ([100, 7, 33], [700, 40, 3]):
        c, table, lengths, t = filled(dev, rng, cache, lens, 16, 2, 64)
        n = sum(lens)
        offs = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64, device=dev)
        k, v = ops.hist_read(c, table, lengths, n, offsets=offs, dtype=torch.float32)
        zero = torch.from_numpy(rng.random((n, 1, 1)) < 0.5).to(dev)
        if power is None:
            v = torch.where(zero, torch.zeros_like(v), v)
            k = torch.where(torch.from_numpy(rng.random((n, 1, 1)) < 0.1).to(dev), torch.zeros_like(k), k)
        else:
            v = v * 2.0 ** power                               # exact in every type
        ops.hist_write(c, k, v, table, lengths, offsets=offs)
        dt = torch.float32 if cache == 'f32' else torch.bfloat16
        q = torch.from_numpy(rng.standard_normal((3, 1, 4, 64))).to(dev, dt)
        got = ops.hist_attn(c, q, table, lengths).double().cpu().numpy()
        want, absv, size = oh.attention(values(c), q.double().cpu().numpy(), t, lens, 0.125, 16)
        held("hist_attn %s rows of zeros / 2^%s, up to %d" % (cache, power, max(lens)),
             (np.abs(got - want) / bound(cache, 64, max(lens), want, absv, size)).max(), 1.0)


@pytest.mark.parametrize('cache', ['bf16', 'e4m3'])
def test_strided_queries_shared_pages_and_table_views(dev, cache):
    """Queries as a slice of a fused projection, several sequences on the same pages, a page table that is a view."""
    from recommendation_amd import ops
    rng = np.random.default_rng(12)
    c, table, lengths, t = filled(dev, rng, cache, [200, 90], 32, 2, 64)
    wide = torch.full((5, 20), -1, dtype=torch.int32, device=dev)
    wide[:, 3:3 + table.shape[1]] = table[torch.tensor([0, 1, 0, 0, 1], device=dev)]
    lens = [200, 90, 150, 1, 33]
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    fused = torch.from_numpy(rng.standard_normal((5, 3 * 8 * 64))).to(dev, torch.bfloat16)
    q = fused[:, 512:1024].view(5, 8, 64)
    view = wide[:, 3:3 + table.shape[1]]
    got = ops.hist_attn(c, q, view, lengths)
    assert got.shape == (5, 8, 64)
    want, absv, size = oh.attention(values(c), q.double().cpu().numpy()[:, None], view.cpu().numpy(), lens, 64 ** -0.5, 32)
    b = bound(cache, 64, 200, want, absv, size)
    held("hist_attn %s strided" % cache, (np.abs(got.double().cpu().numpy()[:, None] - want) / b).max(), 1.0)
    # heads transposed: tokens and heads of a [heads, tokens] tensor
    qt = torch.from_numpy(rng.standard_normal((5, 4, 3, 64))).to(dev, torch.bfloat16).transpose(1, 2)
    got = ops.hist_attn(c, qt, view, lengths)
    want, absv, size = oh.attention(values(c), qt.double().cpu().numpy(), view.cpu().numpy(), lens, 64 ** -0.5, 32)
    held("hist_attn %s transposed" % cache, (np.abs(got.double().cpu().numpy() - want) / bound(cache, 64, 200, want, absv, size)).max(), 1.0)


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
@pytest.mark.parametrize('width', [63, 70])
def test_bad_pages_are_absent_and_reported(dev, cache, width):
    from recommendation_amd import ops
    rng = np.random.default_rng(21)
    lens = [100, 1000, 64, 40]
    c, table, lengths, t = filled(dev, rng, cache, lens, 16, 2, 64, width=width)
    t = t.copy()
    t[0, 2], t[0, 6], t[1, 5], t[1, 30:34] = -1, c.n_pages, 1 << 30, -7
    t[3, :] = -1                                                             # no page at all: zeros
    lens[2] = 64
    dt = torch.float32 if cache == 'f32' else torch.bfloat16
    q = torch.from_numpy(rng.standard_normal((4, 1, 4, 64))).to(dev, dt)
    err = ops.new_error_word(dev)
    got = ops.hist_attn(c, q, torch.from_numpy(t).to(dev), lengths, err=err).double().cpu().numpy()
    want, absv, size = oh.attention(values(c), q.double().cpu().numpy(), t, lens, 64 ** -0.5, 16)
    held("hist_attn %s bad pages" % cache, (np.abs(got - want) / bound(cache, 64, 1000, want, absv, size)).max(), 1.0)
    assert not got[3].any() and err.item() == 1
    # a length beyond the table: its pages' positions only, reported
    err = ops.new_error_word(dev)
    got2 = ops.hist_attn(c, q[2:3], table[2:3, :4], torch.tensor([70], dtype=torch.int32, device=dev), err=err)
    assert err.item() == 1
    # (a narrower table may be summed in another order: held to the definition, not to the call above)
    held("hist_attn %s beyond the table" % cache,
         (np.abs(got2.double().cpu().numpy() - want[2:3]) / bound(cache, 64, 64, want, absv, size)[2:3]).max(), 1.0)
    ops.hist_attn(c, q[2:3], table[2:3, :4], torch.tensor([64], dtype=torch.int32, device=dev), err=ops.new_error_word(dev))


@pytest.mark.parametrize('cache', ['f32', 'bf16'])
def test_infinite_and_nan_values(dev, cache):
    """Rows without a finite score give zeros; an infinite score or a NaN in a live position shows as NaN."""
    from recommendation_amd import ops
    rng = np.random.default_rng(31)
    dt = DTYPES[cache]
    c, table, lengths, t = filled(dev, rng, cache, [40, 40, 40, 40], 16, 1, 64)
    q = torch.from_numpy(rng.standard_normal((4, 1, 1, 64))).to(dev, dt)
    q[:, 0, 0, 0] = 1.0
    clean = ops.hist_attn(c, q, table, lengths)
    page = t[0]
    c.kv[page[:3].tolist(), 0, 0, :, 0] = -float('inf')                      # sequence 0: every score -inf
    c.kv[int(t[1][1]), 0, 0, 5, 0] = -float('inf')                           # sequence 1: one position drops out
    c.kv[int(t[2][2]), 0, 0, 2, 3] = float('nan')                            # sequence 2: a NaN key in a live position
    got = ops.hist_attn(c, q, table, lengths)
    assert not got[0].any()
    assert torch.isnan(got[2]).all()
    assert torch.equal(got[3], clean[3])
    want, absv, size = oh.attention(values(c)[:, :, :, :, :], q.double().cpu().numpy(), t, [0, 40, 0, 0], 0.125, 16)
    size = np.where(np.isfinite(size), size, 64.0)
    err = (np.abs(got[1].double().cpu().numpy() - want[1]) / bound(cache, 64, 40, want, absv, size)[1]).max()
    held("hist_attn %s one -inf score" % cache, err, 1.0)


@pytest.mark.parametrize('dim', [32, 128])
@pytest.mark.parametrize('lens', [[40, 40, 40, 40], [700, 40, 600, 700], [1500, 40, 1400, 1500]])
def test_nan_codes_in_an_8_bit_cache(dev, lens, dim):
    """Written as infinities and NaN: a NaN in a live key makes the row's result NaN, one in a live value its channel; behind
    the history, in dead slots of the last page, neither they nor exponent bytes of 255 are seen."""
    from recommendation_amd import ops
    rng = np.random.default_rng(33)
    c, table, lengths, t = filled(dev, rng, 'e4m3', lens, 16, 2, dim)
    q = torch.from_numpy(rng.standard_normal((4, 1, 4, dim))).to(dev, torch.bfloat16)
    clean = ops.hist_attn(c, q, table, lengths)
    assert torch.isfinite(clean).all()                                       # the rest of the cache is NaN
    offs = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64, device=dev)
    k, v = ops.hist_read(c, table, lengths, sum(lens), offsets=offs, dtype=torch.float32)
    at = np.concatenate([[0], np.cumsum(lens)])
    k[int(at[1]) + 21, 0, 5] = float('inf')                                  # user 1, head 0: a key
    v[int(at[2]) + lens[2] - 1, 1, 7] = float('nan')                         # user 2, head 1: channel 7 of the newest value
    v[int(at[2]) + 3, 1, 9] = -float('inf')
    ops.hist_write(c, k, v, table, lengths, offsets=offs)
    got = ops.hist_attn(c, q, table, lengths)
    want = clean.clone()
    want[1, :, :2] = float('nan')
    want[2, :, 2:, 7] = want[2, :, 2:, 9] = float('nan')
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    keep = ~torch.isnan(want)
    assert torch.equal(got[keep], clean[keep])
    shorter = lengths - torch.tensor([0, 20, 1, 0], dtype=torch.int32, device=dev)   # user 2's newest row is dead now
    got = ops.hist_attn(c, q, table, shorter)
    assert not torch.isnan(got[1]).any() and not torch.isnan(got[2, :, :, 7]).any() and torch.isnan(got[2, :, 2:, 9]).all()


@pytest.mark.parametrize('cache', ['f32', 'bf16'])
@pytest.mark.parametrize('lens', [[40, 33], [700, 600], [1500, 1300]])
def test_an_infinite_score_shows_as_nan(dev, cache, lens):
    """+inf - +inf: the whole result of that query head is NaN, early or late in the history, the other user's is not touched."""
    from recommendation_amd import ops
    rng = np.random.default_rng(34)
    c, table, lengths, t = filled(dev, rng, cache, lens, 16, 1, 64)
    q = torch.from_numpy(rng.standard_normal((2, 1, 2, 64))).to(dev, DTYPES[cache])
    q[:, :, :, 0] = 1.0
    clean = ops.hist_attn(c, q, table, lengths)
    for pos in (0, 17, lens[0] - 1):
        held_key = c.kv[int(t[0][pos // 16]), 0, 0, pos % 16, 0].clone()
        c.kv[int(t[0][pos // 16]), 0, 0, pos % 16, 0] = float('inf')
        got = ops.hist_attn(c, q, table, lengths)
        assert torch.isnan(got[0]).all() and torch.equal(got[1], clean[1])
        c.kv[int(t[0][pos // 16]), 0, 0, pos % 16, 0] = held_key
    assert torch.equal(ops.hist_attn(c, q, table, lengths), clean)


# ------------------------------------------------------------------------------------------------ used together
@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
def test_histories_grow_event_by_event(dev, cache):
    """The serving loop: prompts in one call, then one event a step for a batch in which some users pause (length 0),
    attention after each; captured once and replayed on new inputs, equal to the eager calls bit for bit."""
    from recommendation_amd import ops
    rng = np.random.default_rng(5)
    dt = torch.float32 if cache == 'f32' else torch.bfloat16
    heads, group, dim, page, users, width = 2, 3, 64, 16, 6, 6
    c = poisoned(dev, cache, users * width, page, heads, dim)
    twin = poisoned(dev, cache, users * width, page, heads, dim)
    table = torch.from_numpy(rng.permutation(users * width).astype(np.int32).reshape(users, width)).to(dev)
    start = np.array([0, 14, 15, 16, 31, 50])
    offs = np.concatenate([[0], np.cumsum(start)]).astype(np.int64)
    rows = torch.from_numpy(rng.standard_normal((int(offs[-1]), 2, heads, dim))).to(dev, dt)
    lens = torch.from_numpy(start.astype(np.int32)).to(dev)
    for x in (c, twin):
        ops.hist_write(x, rows[:, 0], rows[:, 1], table, lens, offsets=torch.from_numpy(offs).to(dev))
    k, v = (torch.zeros((users, heads, dim), dtype=dt, device=dev) for _ in range(2))
    q = torch.zeros((users, heads * group, dim), dtype=dt, device=dev)
    step_lens = lens.clone()
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                                            # a length of 0 pauses everybody: no effect
        zero = torch.zeros_like(lens)
        ops.hist_write(c, k, v, table, zero)
        ops.hist_attn(c, q, table, zero, out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert not out.any()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.hist_write(c, k, v, table, step_lens)
        ops.hist_attn(c, q, table, step_lens, out=out)
    held_len = start.copy()
    for step in range(20):
        k.copy_(torch.from_numpy(rng.standard_normal(tuple(k.shape))))
        v.copy_(torch.from_numpy(rng.standard_normal(tuple(k.shape))))
        q.copy_(torch.from_numpy(rng.standard_normal(tuple(q.shape))))
        paused = rng.random(users) < 0.3
        held_len = held_len + ~paused
        now = np.where(paused, 0, held_len).astype(np.int32)
        step_lens.copy_(torch.from_numpy(now))
        graph.replay()
        ops.hist_write(twin, k, v, table, step_lens)
        eager = ops.hist_attn(twin, q, table, step_lens)
        assert torch.equal(out, eager)
        assert not out[torch.from_numpy(paused).to(dev)].any()
    np.testing.assert_array_equal(values(c), values(twin))
    final = torch.from_numpy(held_len.astype(np.int32)).to(dev)
    got = ops.hist_attn(c, q, table, final).double().cpu().numpy()[:, None]
    want, absv, size = oh.attention(values(c), q.double().cpu().numpy()[:, None], table.cpu().numpy(), held_len, dim ** -0.5, page)
    held("hist_attn %s grown" % cache, (np.abs(got - want) / bound(cache, dim, 80, want, absv, size)).max(), 1.0)
    # the histories read back and written into a fresh cache are the same histories
    total = int(held_len.sum())
    offs = torch.from_numpy(np.concatenate([[0], np.cumsum(held_len)]).astype(np.int64)).to(dev)
    k2, v2 = ops.hist_read(c, table, final, total, offsets=offs, dtype=torch.float32)
    fresh = poisoned(dev, cache, users * width, page, heads, dim)
    ops.hist_write(fresh, k2, v2, table, final, offsets=offs)
    np.testing.assert_array_equal(values(fresh), values(c))


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
@pytest.mark.parametrize('before', [3, 600, 3000])
def test_several_events_of_one_user_see_those_before_them(dev, cache, before):
    """Events appended in one call, each attending up to itself: one sequence per event over the user's expanded table row."""
    from recommendation_amd import ops
    rng = np.random.default_rng(before)
    page, heads, dim, new = 16, 2, 64, 5
    total = before + new
    c, table, lengths, t = filled(dev, rng, cache, [total], page, heads, dim)
    k, v = (torch.from_numpy(rng.integers(-7, 8, size=(new, heads, dim))).to(dev, torch.float32) for _ in range(2))
    ops.hist_write(c, k, v, table, lengths)                                  # whole numbers: exact in every type
    dt = torch.float32 if cache == 'f32' else torch.bfloat16
    q = torch.from_numpy(rng.standard_normal((new, 4, dim))).to(dev, dt)
    rows = table.expand(new, -1)
    lens = np.arange(before + 1, total + 1)
    upto = torch.from_numpy(lens.astype(np.int32)).to(dev)
    got = ops.hist_attn(c, q, rows, upto)
    assert torch.equal(got, ops.hist_attn(c, q, rows.contiguous(), upto))
    want, absv, size = oh.attention(values(c), q.double().cpu().numpy()[:, None], np.repeat(t, new, 0), lens, dim ** -0.5, page)
    held("hist_attn %s events of one user after %d" % (cache, before),
         (np.abs(got.double().cpu().numpy()[:, None] - want) / bound(cache, dim, total, want, absv, size)).max(), 1.0)
    k2, v2 = ops.hist_read(c, rows, upto, new, dtype=torch.float32)          # each event's own row
    assert torch.equal(k2, k) and torch.equal(v2, v)
    with pytest.raises(ops.MiError, match='row stride'):
        ops.hist_write(c, k, v, rows, upto)


def test_captured_attention_over_long_histories(dev):
    """The two launches and the workspace between them inside graphs: two graphs captured one after the other, replayed in
    turn on two streams with new lengths and queries, eager calls between; every replay equals the eager call."""
    from recommendation_amd import ops
    rng = np.random.default_rng(14)
    c, table, lengths, t = filled(dev, rng, 'bf16', [3000, 2900, 1, 600, 0], 16, 2, 128)
    full = lengths.clone()
    qs = [torch.from_numpy(rng.standard_normal((5, 8, 128))).to(dev, torch.bfloat16) for _ in range(2)]
    outs = [torch.zeros_like(q) for q in qs]
    lens = [full.clone(), full.clone()]
    ops.hist_attn(c, qs[0], table, full)
    torch.cuda.synchronize()
    graphs = []
    for q, out, n in zip(qs, outs, lens):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.hist_attn(c, q, table, n, out=out)
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for step in range(6):
        for i in range(2):
            qs[i].copy_(torch.from_numpy(rng.standard_normal((5, 8, 128))))
            lens[i].copy_(torch.clamp(full - int(rng.integers(0, 500)), min=0))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        eager = [ops.hist_attn(c, qs[i], table, lens[i]) for i in range(2)]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1])
        assert not eager[0][4].any()


def test_the_result_may_replace_the_queries(dev):
    from recommendation_amd import ops
    rng = np.random.default_rng(15)
    for lens in ([50, 3, 0], [600, 3, 0], [4000, 70, 900]):
        c, table, lengths, t = filled(dev, rng, 'e4m3', lens, 16, 2, 64)
        q = torch.from_numpy(rng.standard_normal((3, 20, 6, 64))).to(dev, torch.bfloat16)
        want = ops.hist_attn(c, q, table, lengths)
        assert ops.hist_attn(c, q, table, lengths, out=q) is q and torch.equal(q, want)


@pytest.mark.parametrize('cache', ['f32', 'bf16', 'e4m3'])
def test_results_between_each_other_and_between_the_queries(dev, cache):
    """Results that lie in one buffer with each other or with the queries, and share no row: interleaved by token, by head, heads
    in front, with gaps of different width."""
    from recommendation_amd import ops
    rng = np.random.default_rng(41)
    heads, dim, lens = 2, 64, [40, 0, 100]
    n, dt = sum(lens), torch.float32 if cache == 'f32' else torch.bfloat16
    c, table, lengths, t = filled(dev, rng, cache, lens, 16, heads, dim)
    offs = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int64, device=dev)
    k, v = ops.hist_read(c, table, lengths, n, offsets=offs, dtype=dt)
    new = lambda *shape: torch.full(shape, 5.0, dtype=dt, device=dev)
    a, b, d, e = new(n, 2, heads, dim), new(n, heads, 2, dim), new(2, heads, n, dim), new(n, 2 * heads * dim + heads * 16)
    half = heads * dim
    for pair in ((a[:, 0], a[:, 1]), (b[:, :, 1], b[:, :, 0]), (d[0].transpose(0, 1), d[1].transpose(0, 1)),
                 (e[:, :half].view(n, heads, dim), e[:, half:].view(n, heads, dim + 16)[..., :dim])):
        ops.hist_read(c, table, lengths, offsets=offs, out=pair)
        assert torch.equal(pair[0], k) and torch.equal(pair[1], v)
    assert bool((e[:, half:].view(n, heads, dim + 16)[..., dim:] == 5.0).all())
    q = torch.from_numpy(rng.standard_normal((3, 2, 4, dim))).to(dev, dt)
    want = ops.hist_attn(c, q, table, lengths)
    a, b, d = new(3, 2, 2, 4, dim), new(3, 2, 4, 2, dim), new(3, 4, 2, 2 * dim)
    views = [(a[:, :, 0], a[:, :, 1]), (a[:, 1], a[:, 0]), (b[..., 1, :], b[..., 0, :]),
             (d[..., :dim].transpose(1, 2), d[..., dim:].transpose(1, 2))]
    for mine, out in views:
        mine.copy_(q)
        ops.hist_attn(c, mine, table, lengths, out=out)
        assert torch.equal(out, want) and torch.equal(mine, q)
    x = new(3, 4, 2, dim).transpose(1, 2)
    x.copy_(q)
    assert ops.hist_attn(c, x, table, lengths, out=x) is x and torch.equal(x, want)
    for bad in (lambda: ops.hist_read(c, table, lengths, offsets=offs, out=(k, k)),
                lambda: ops.hist_attn(c, q, table, lengths, out=q.view(3, 4, 2, dim).transpose(1, 2))):
        with pytest.raises(ops.MiError, match='overlap'):
            bad()


def test_two_calls_at_once_on_two_streams(dev):
    """Calls that share nothing but the cache they read run side by side with their own workspaces."""
    from recommendation_amd import ops
    rng = np.random.default_rng(6)
    c, table, lengths, t = filled(dev, rng, 'bf16', [9000, 100, 4000], 16, 2, 64)
    qs = [torch.from_numpy(rng.standard_normal((3, 8, 64))).to(dev, torch.bfloat16) for _ in range(2)]
    want = [ops.hist_attn(c, q, table, lengths) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.hist_attn(c, qs[i], table, lengths))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_offsets_into_a_pool_past_32_bits(dev):
    """Pages whose bytes, and element indexes, lie past 2^32."""
    from recommendation_amd import ops
    rng = np.random.default_rng(8)
    page, heads, dim = 1024, 8, 256
    n_pages = (1 << 33) // (heads * 2 * page * dim) + 5                       # 2^33 elements of 8 bits
    kv = torch.empty((n_pages, heads, 2, page, dim), dtype=torch.uint8, device=dev)
    kv[-4:].fill_(0x7f)
    c = ops.HistCache(n_pages, page, heads, dim, dtype=torch.float8_e4m3fn, kv=kv.view(torch.float8_e4m3fn))
    table = torch.tensor([[n_pages - 1, n_pages - 3], [n_pages - 2, -1]], dtype=torch.int32, device=dev)
    lens = [1100, 3]
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)
    offs = torch.tensor([0, 1100, 1103], dtype=torch.int64, device=dev)
    rows = torch.from_numpy(rng.standard_normal((1103, 2, heads, dim))).to(dev, torch.bfloat16)
    ops.hist_write(c, rows[:, 0], rows[:, 1], table, lengths, offsets=offs)
    k, v = ops.hist_read(c, table, lengths, 1103, offsets=offs, dtype=torch.float32)
    held_rows = oh.quantise(rows.double().cpu().numpy())[0]
    np.testing.assert_array_equal(k.cpu().numpy(), held_rows[:, 0].astype(np.float32))
    np.testing.assert_array_equal(v.cpu().numpy(), held_rows[:, 1].astype(np.float32))
    q = torch.from_numpy(rng.standard_normal((2, 1, heads, dim))).to(dev, torch.bfloat16)
    got = ops.hist_attn(c, q, table, lengths).double().cpu().numpy()
    small = np.zeros((3, heads, 2, page, dim))
    small[0, :, 0], small[0, :, 1] = held_rows[:1024, 0].transpose(1, 0, 2), held_rows[:1024, 1].transpose(1, 0, 2)
    small[1, :, 0, :76], small[1, :, 1, :76] = held_rows[1024:1100, 0].transpose(1, 0, 2), held_rows[1024:1100, 1].transpose(1, 0, 2)
    small[2, :, 0, :3], small[2, :, 1, :3] = held_rows[1100:, 0].transpose(1, 0, 2), held_rows[1100:, 1].transpose(1, 0, 2)
    want, absv, size = oh.attention(small, q.double().cpu().numpy(), np.array([[0, 1], [2, -1]]), lens, dim ** -0.5, page)
    held("hist_attn past 2^32", (np.abs(got - want) / bound('e4m3', dim, 1100, want, absv, size)).max(), 1.0)


# ------------------------------------------------------------------------------------------------ refusals
def test_calls_that_do_not_fit_are_refused(dev):
    from recommendation_amd import ops
    c = ops.HistCache(8, 16, 2, 64, device=dev)
    c.kv.zero_()
    table = torch.zeros((3, 2), dtype=torch.int32, device=dev)
    lengths = torch.zeros(3, dtype=torch.int32, device=dev)
    k = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device=dev)
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device=dev)
    for bad, exc, text in [
            (lambda: ops.hist_write(c, k.half(), k.half(), table, lengths), TypeError, 'float32 or bfloat16'),
            (lambda: ops.hist_write(c, k, k.float(), table, lengths), ops.MiError, 'differ'),
            (lambda: ops.hist_write(c, k[:, :1], k[:, :1], table, lengths), ops.MiError, 'rows must be'),
            (lambda: ops.hist_write(c, k[:2], k[:2], table, lengths), ops.MiError, 'divide'),
            (lambda: ops.hist_write(c, k, k, table.long(), lengths), ops.MiError, 'page_table'),
            (lambda: ops.hist_write(c, k, k, table.t(), lengths), ops.MiError, 'page_table'),
            (lambda: ops.hist_write(c, k, k, table, lengths.long()), ops.MiError, 'lengths'),
            (lambda: ops.hist_write(c, k, k, table, lengths[:2]), ops.MiError, 'lengths'),
            (lambda: ops.hist_write(c, k, k, table, lengths, offsets=lengths), ops.MiError, 'offsets'),
            (lambda: ops.hist_write(c, k.cpu(), k.cpu(), table, lengths), ops.MiError, 'device tensors'),
            (lambda: ops.hist_write(c, k.transpose(1, 2).contiguous().transpose(1, 2), k, table, lengths), ops.MiError, 'contiguous'),
            (lambda: ops.hist_write(c, torch.zeros(3 * 128 + 4, dtype=torch.bfloat16, device=dev)[4:].view(3, 2, 64), k, table, lengths),
             ops.MiError, '16-byte'),
            (lambda: ops.hist_read(c, table, lengths), ops.MiError, 'n_rows'),
            (lambda: ops.hist_read(c, table, lengths, 3, dtype=torch.float16), TypeError, 'float32 or bfloat16'),
            (lambda: ops.hist_read(c, table, lengths, 4, out=(k, k.clone())), ops.MiError, 'n_rows'),
            (lambda: ops.hist_attn(c, q.float(), table, lengths), TypeError, 'bfloat16'),
            (lambda: ops.hist_attn(c, q[:, :3], table, lengths), ops.MiError, 'multiple'),
            (lambda: ops.hist_attn(c, q[:2], table, lengths), ops.MiError, 'q must be'),
            (lambda: ops.hist_attn(c, q, table, lengths, out=q.float()), ops.MiError, 'out'),
            (lambda: ops.hist_attn(c, q, table, lengths, err=torch.zeros(1, device=dev)), ops.MiError, 'err'),
            (lambda: ops.HistCache(8, 16, 2, 64, kv=c.kv[:4]), ops.MiError, 'kv must be'),
            (lambda: ops.HistCache(8, 16, 2, 64, kv=c.kv, exps=torch.zeros((8, 2, 2, 16), dtype=torch.uint8, device=dev)), ops.MiError, 'exps'),
            (lambda: ops.HistCache(8, 16, 2, 64, dtype=torch.float8_e4m3fn, device=dev, kv=None,
                                   exps=torch.zeros((8, 2, 2, 16), dtype=torch.uint8, device=dev)), ops.MiError, 'exps')]:
        with pytest.raises(exc, match=text):
            bad()
    # nothing to do
    ops.hist_write(c, k[:0], k[:0], table[:0], lengths[:0])
    assert ops.hist_attn(c, q[:0], table[:0], lengths[:0]).shape == (0, 4, 64)
    assert ops.hist_attn(c, q.view(3, 1, 4, 64)[:, :0], table, lengths).shape == (3, 0, 4, 64)
    assert ops.hist_read(c, table, lengths, 0)[0].shape == (0, 2, 64)
