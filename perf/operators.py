"""Cases that the history-cache operators are measured on: rows of keys and values appended to the users' pages
(hist_write), read back (hist_read) and attended by new tokens or candidates (hist_attn).

Each case runs in two forms: the plain one (elementary torch operations in 32 bits) and, where ``own`` is set, the
framework's entry points in ``recommendation_amd.ops``.  Cache layout of both: kv [n_pages, heads, 2, page_size, dim]
(0 keys, 1 values) and, for 8-bit caches, exps [n_pages, heads, 2, page_size] (a row stands for code * 2^(exps - 127)).
"""
import math

import torch

own = False

_TORCH = {'f32': torch.float32, 'bf16': torch.bfloat16, 'e4m3': torch.float8_e4m3fn}
_BYTES = {'f32': 4, 'bf16': 2, 'e4m3': 1}


# ----------------------------------------------------------------------------- cases
def _attn(name, cache, users, queries, q_heads, heads, dim, page, shortest, longest, spread):
    """Attention of `queries` new tokens (or candidates) of each user over the user's history.  spread: 'even' lengths
    are uniform in [shortest, longest], 'log' lengths uniform in their logarithm with one user at the longest."""
    return dict(name=name, op='attn', cache=cache, users=users, queries=queries, q_heads=q_heads, heads=heads, dim=dim,
                page=page, shortest=shortest, longest=longest, spread=spread)


def _rows(name, op, cache, given, users, heads, dim, page, rows, longest):
    """`rows` rows of K and V in all, spread over the users' newest positions; histories up to `longest` rows."""
    return dict(name=name, op=op, cache=cache, given=given, users=users, heads=heads, dim=dim, page=page, rows=rows,
                longest=longest)


def listed():
    return [
        # one user, one candidate, a history of 100 events (the DIN unit's history length and width): latency alone
        _attn('attn_one_user', 'bf16', 1, 1, 8, 8, 64, 16, 100, 100, 'even'),
        # the DIN batch: 8192 samples, histories of up to 100 events (empty ones among them), one head of width 64
        _attn('attn_din_batch', 'bf16', 8192, 1, 1, 1, 64, 16, 0, 100, 'even'),
        # a serving batch of 300 users in 32 bits, narrow heads, lengths from a few events to some thousands
        _attn('attn_serving_f32', 'f32', 300, 1, 4, 4, 32, 16, 1, 2000, 'log'),
        # few users with long histories in 8 bits, four query heads to a cache head: the length has to be split
        _attn('attn_long_e4m3', 'e4m3', 16, 1, 32, 8, 128, 64, 16000, 32768, 'even'),
        # many users, one of them with a very long history: work per user differs a thousandfold
        _attn('attn_ragged_bf16', 'bf16', 64, 1, 16, 2, 128, 16, 1, 100000, 'log'),
        # ranking: 16 candidates a user against the same history
        _attn('attn_candidates_e4m3', 'e4m3', 32, 16, 8, 2, 128, 32, 300, 8191, 'even'),
        # the largest: 64 users, 8,000 to 16,000 events each, bf16
        _attn('attn_large_bf16', 'bf16', 64, 1, 32, 8, 128, 64, 8000, 16384, 'even'),
        # one event for each of 300 users appended to an 8-bit cache and read back: latency
        _rows('write_events_e4m3', 'write', 'e4m3', 'bf16', 300, 4, 64, 16, 300, 3000),
        # whole histories of 509 users cached in 8 bits, and read back
        _rows('write_histories_e4m3', 'write', 'e4m3', 'bf16', 509, 8, 128, 32, 65521, 600),
        # histories in a 16-bit cache, computed in 32 bits
        _rows('write_histories_bf16', 'write', 'bf16', 'f32', 64, 4, 64, 16, 20011, 1000),
        # a few users' newest events read back in 32 bits
        _rows('read_events_f32', 'read', 'e4m3', 'f32', 3, 8, 64, 16, 257, 1500),
        # long histories read back in 16 bits
        _rows('read_histories_bf16', 'read', 'e4m3', 'bf16', 64, 8, 128, 64, 250007, 8000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['attn', 'attn', 'attn', 'write', 'read'])
    cache = rng.choice(['f32', 'bf16', 'bf16', 'e4m3', 'e4m3'])
    dim = rng.choice([32, 64, 64, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64, 128])
    heads = rng.choice([1, 2, 4, 8])
    users = _log(rng, 1, 8192)
    row_bytes = 2 * heads * dim * _BYTES[cache]
    if op == 'attn':
        group = rng.choice([1, 1, 2, 3, 4, 7, 8])
        queries = rng.choice([1, 1, 1, 2, 5, 16])
        longest = max(1, min(_log(rng, 30, 100000), int(1.2e9 / (users * row_bytes)),
                             int(3e8 / (users * heads * dim)),
                             int(2.4e9 / (users * queries * heads * group * dim))))
        case = _attn('', cache, users, queries, heads * group, heads, dim, page, rng.choice([0, 1, longest // 2]), longest,
                     rng.choice(['even', 'log']))
    else:
        rows = max(users, min(_log(rng, 1, 250000), int(4e8 / (heads * dim * 8))))
        given = 'f32' if cache == 'f32' else rng.choice(['f32', 'bf16', 'bf16'])
        longest = max(-(-rows // users) * 2, min(8000, int(5e8 / (users * row_bytes))))
        case = _rows('', op, cache, given, users, heads, dim, page, rows, longest)
    del case['name']
    return case


# ----------------------------------------------------------------------------- inputs
def _lengths(case, gen):
    """(history lengths, rows of each user that this call writes or reads), as lists: a program that plans its batch
    has them on the host."""
    n = case['users']
    u = torch.rand(n, generator=gen, dtype=torch.float64)
    if case['op'] == 'attn':
        lo, hi = case['shortest'], case['longest']
        if case['spread'] == 'log':
            lens = torch.exp(u * math.log((hi + 1) / max(lo, 1)) + math.log(max(lo, 1))).long()
            lens[int(torch.randint(n, (1,), generator=gen))] = hi
        else:
            lens = lo + (u * (hi - lo + 1)).long()
        return lens.clamp(max=hi).tolist(), None
    # rows per user: uneven, summing to the case's total, each at most `longest`
    total, cap = case['rows'], case['longest']
    if total == n:
        rows = [1] * n
    else:
        w = u + 0.25
        rows = torch.clamp((w / w.sum() * total).long(), max=cap).tolist()
        left, i = total - sum(rows), 0
        while left:
            more = min(left, cap - rows[i], 1 + left // n)
            rows[i] += more
            left -= more
            i = (i + 1) % n
    more = torch.rand(n, generator=gen, dtype=torch.float64)
    return [r + int(m * (cap - r + 1)) for r, m in zip(rows, more.tolist())], rows


def _two_to(e):
    """2^e as float32 for int32 tensors of exponents in [-126, 127]."""
    return ((e + 127) << 23).view(torch.float32)


def _quantised(x):
    """codes and exponent bytes of rows x [..., dim], float32."""
    top = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1)
    m, e = torch.frexp(top)                                   # top = m * 2^e, m in [0.5, 1)
    e = e.to(torch.int32) - 9 + (m > 0.875).to(torch.int32)    # the smallest e with top * 2^-e <= 448
    e = torch.where(top > 0, e, torch.full_like(e, -126)).clamp(min=-126)
    codes = (x * _two_to(-e)[..., None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _values(codes, exps):
    if exps is None:
        return codes.float()
    return codes.float() * _two_to(exps.to(torch.int32) - 127)[..., None]


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev = torch.device('cuda')
    rnd = torch.Generator(device=dev).manual_seed(seed)
    lens, rows = _lengths(case, gen)
    users, heads, dim, page, cache = case['users'], case['heads'], case['dim'], case['page'], case['cache']
    width = max(1, -(-max(max(lens), 1) // page))
    used = [-(-n // page) for n in lens]
    # the pool of a write case is an output: its size goes by the case alone
    n_pages = users * -(-case['longest'] // page) if case['op'] == 'write' else sum(used) + 3
    order = torch.randperm(n_pages, generator=gen, dtype=torch.int64).to(torch.int32)
    table = torch.full((users, width), -1, dtype=torch.int32)
    at = 0
    for b, k in enumerate(used):
        table[b, :k] = order[at:at + k]
        at += k
    shape = (n_pages, heads, 2, page, dim)
    exps = None
    if case['op'] == 'write':
        kv = torch.zeros(shape, dtype=torch.uint8 if cache == 'e4m3' else _TORCH[cache], device=dev)
        if cache == 'e4m3':
            kv, exps = kv.view(_TORCH[cache]), torch.zeros(shape[:-1], dtype=torch.uint8, device=dev)
    else:
        kv = torch.empty(shape, dtype=_TORCH[cache], device=dev)
        if cache == 'e4m3':
            exps = torch.empty(shape[:-1], dtype=torch.uint8, device=dev)
        step = max(1, (1 << 27) // (heads * 2 * page * dim))
        for i in range(0, n_pages, step):
            part = torch.randn((min(step, n_pages - i),) + shape[1:], generator=rnd, device=dev)
            if exps is None:
                kv[i:i + step] = part.to(_TORCH[cache])
            else:
                codes, e = _quantised(part)
                kv.view(torch.uint8)[i:i + step] = codes.view(torch.uint8)
                exps[i:i + step] = e
    st = dict(case=case, lens=lens, rows=rows, kv=kv, exps=exps, table=table.to(dev),
              lengths=torch.tensor(lens, dtype=torch.int32, device=dev))
    if case['op'] == 'attn':
        # scores with a few high ones, as a trained model's are
        q = torch.randn((users, case['queries'], case['q_heads'], dim), generator=rnd, device=dev) * 1.5
        st['q'] = q.to(torch.float32 if cache == 'f32' else torch.bfloat16)
    else:
        offs = [0]
        for r in rows:
            offs.append(offs[-1] + r)
        st['offs'] = offs
        st['offsets'] = torch.tensor(offs, dtype=torch.int64, device=dev)
        if case['op'] == 'write':
            # K and V side by side, as one projection leaves them; rows of very different size
            kvrows = torch.randn((offs[-1], 2, heads, dim), generator=rnd, device=dev)
            kvrows *= torch.exp2(4 * torch.randn((offs[-1], 2, heads, 1), generator=rnd, device=dev))
            kvrows = kvrows.to(_TORCH[case['given']])
            st['k'], st['v'] = kvrows[:, 0], kvrows[:, 1]
    if own:
        from recommendation_amd import ops
        st['cache'] = ops.HistCache(n_pages, page, heads, dim, dtype=_TORCH[cache], kv=kv, exps=exps)
    return st


# ----------------------------------------------------------------------------- one pass
def _places(st):
    """Page and slot of every row that a write or read call covers."""
    case = st['case']
    offsets, lengths = st['offsets'], st['lengths'].long()
    i = torch.arange(st['offs'][-1], device=offsets.device)
    b = torch.searchsorted(offsets, i, right=True) - 1
    pos = lengths[b] - (offsets[b + 1] - i)
    return st['table'].long()[b, pos // case['page']], pos % case['page']


def _plain_write(st):
    page, slot = _places(st)
    kv, exps = st['kv'], st['exps']
    for part, x in ((0, st['k']), (1, st['v'])):
        if exps is None:
            kv[page, :, part, slot] = x.to(kv.dtype)
        else:
            codes, e = _quantised(x.float())
            kv.view(torch.uint8)[page, :, part, slot] = codes.view(torch.uint8)
            exps[page, :, part, slot] = e


def _plain_read(st, dtype):
    page, slot = _places(st)
    kv, exps = st['kv'], st['exps']
    out = []
    for part in (0, 1):
        if exps is None:
            x = kv[page, :, part, slot].float()
        else:
            x = _values(kv.view(torch.uint8)[page, :, part, slot].view(kv.dtype), exps[page, :, part, slot])
        out.append(x.to(dtype))
    return tuple(out)


def _plain_attn(st):
    case = st['case']
    users, heads, dim, page = case['users'], case['heads'], case['dim'], case['page']
    kv, exps, q = st['kv'], st['exps'], st['q']
    longest = st['table'].shape[1] * page
    group = case['q_heads'] // heads
    out = torch.empty_like(q)
    step = max(1, (1 << 31) // (longest * heads * dim))
    for lo in range(0, users, step):
        table = st['table'][lo:lo + step].long().clamp(min=0)
        n = table.shape[0]
        live = torch.arange(longest, device=q.device)[None, :] < st['lengths'][lo:lo + step, None]

        def rows(part):
            if exps is None:
                x = kv[:, :, part][table].float()
            else:
                x = _values(kv.view(torch.uint8)[:, :, part][table].view(kv.dtype), exps[:, :, part][table])
            return x.transpose(1, 2).reshape(n, heads, longest, dim)

        qs = q[lo:lo + step].float().view(n, case['queries'], heads, group, dim).permute(0, 2, 1, 3, 4)
        s = torch.matmul(qs.reshape(n, heads, -1, dim), rows(0).transpose(2, 3).contiguous()) / math.sqrt(dim)
        s = torch.where(live[:, None, None, :], s, torch.full_like(s, -math.inf))
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, rows(1)) / torch.where(total == 0, torch.ones_like(total), total)
        o = o.view(n, heads, case['queries'], group, dim).permute(0, 2, 1, 3, 4)
        out[lo:lo + step] = o.reshape(n, case['queries'], case['q_heads'], dim).to(out.dtype)
    return out


def run(st):
    case = st['case']
    given = _TORCH[case['given']] if 'given' in case else None
    if own:
        from recommendation_amd import ops
        if case['op'] == 'attn':
            return ops.hist_attn(st['cache'], st['q'], st['table'], st['lengths'])
        if case['op'] == 'read':
            return ops.hist_read(st['cache'], st['table'], st['lengths'], st['offs'][-1], offsets=st['offsets'], dtype=given)
        ops.hist_write(st['cache'], st['k'], st['v'], st['table'], st['lengths'], offsets=st['offsets'])
        if case['cache'] != 'e4m3':
            return st['kv']
        # 8-bit rows are returned as the values they stand for
        return ops.hist_read(st['cache'], st['table'], st['lengths'], st['offs'][-1], offsets=st['offsets'],
                             dtype=torch.float32)
    if case['op'] == 'attn':
        return _plain_attn(st)
    if case['op'] == 'read':
        return _plain_read(st, given)
    _plain_write(st)
    return st['kv'] if case['cache'] != 'e4m3' else _plain_read(st, torch.float32)


# ----------------------------------------------------------------------------- work
def work(case):
    e = _BYTES[case['cache']]
    row = 2 * case['heads'] * (case['dim'] * e + (1 if case['cache'] == 'e4m3' else 0))     # K and V of one position
    users = case['users']
    if case['op'] == 'attn':
        lo, hi = case['shortest'], case['longest']
        if case['spread'] == 'log':
            first = max(lo, 1)
            mean = (hi + 1 - first) / math.log((hi + 1) / first)
            total = mean * (users - 1) + hi
        else:
            total = (lo + hi) / 2 * users
        pages = total / case['page'] + users / 2
        q = users * case['queries'] * case['q_heads'] * case['dim'] * (4 if case['cache'] == 'f32' else 2)
        return {"bytes": int(total * row + 2 * q + 4 * pages + 4 * users),
                "flops": int(4 * case['dim'] * case['queries'] * case['q_heads'] * total)}
    rows = case['rows']
    values = 2 * case['heads'] * case['dim'] * rows
    index = 12 * users + 4 * (rows // case['page'] + users)
    if case['op'] == 'read':
        return {"bytes": rows * row + values * _BYTES[case['given']] + index, "flops": values}
    moved = values * _BYTES[case['given']] + rows * row + index
    if case['cache'] == 'e4m3':
        moved += rows * row + values * 4 + index                 # read back
    return {"bytes": moved, "flops": 2 * values}


# ----------------------------------------------------------------------------- the definition in 64 bits
def _row_index(st, b, first, last):
    """Flat [page, slot] positions first..last-1 of user b, from the table on the host."""
    page = st['case']['page']
    pos = torch.arange(first, last)
    return st['host_table'][b][pos // page].long().to('cuda'), (pos % page).to('cuda')


def _pow2(e):
    """2^e in 64 bits for whole e in [-1022, 1023], from its bits (a library's pow() may be one unit off)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _floor_log2(x):
    """floor(log2 x) of normal positive 64-bit x."""
    return (x.view(torch.int64) >> 52) - 1023


def _wide(st, pages, slots, part):
    """Rows [positions, heads, dim] of the cache in 64 bits."""
    kv, exps = st['kv'], st['exps']
    if exps is None:
        return kv[pages, :, part, slots].double()
    bits = kv.view(torch.uint8)[pages, :, part, slots].long()
    sign = 1.0 - 2.0 * (bits >> 7).double()
    field, frac = (bits >> 3) & 15, (bits & 7).double()
    mag = torch.where(field == 0, frac * 2.0 ** -9, (8 + frac) * _pow2(field - 10))
    return sign * mag * _pow2(exps[pages, :, part, slots].long() - 127)[..., None]


def _wide_quantised(x):
    """What rows x (64 bits, finite) stand for once they are held in 8 bits."""
    top = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -200)
    power = _floor_log2(top)
    scale = _pow2(torch.clamp(power - 8 + (top > 1.75 * _pow2(power)).long(), min=-126))
    y = x / scale
    step = _pow2(_floor_log2(torch.clamp(y.abs(), min=2.0 ** -6)) - 3)
    return torch.round(y / step) * step * scale                  # round() takes ties to even


def exact(case, seed):
    st = prepare(case, seed)
    st['host_table'] = st['table'].cpu()
    if case['op'] == 'attn':
        q = st['q'].double()
        out = torch.zeros_like(q)
        group = case['q_heads'] // case['heads']
        if case['users'] <= 512:
            for b, n in enumerate(st['lens']):
                if n == 0:
                    continue
                pages, slots = _row_index(st, b, 0, n)
                k = _wide(st, pages, slots, 0).transpose(0, 1).repeat_interleave(group, 0)      # [q_heads, n, dim]
                s = torch.matmul(k, q[b].permute(1, 2, 0).contiguous()).transpose(1, 2) / math.sqrt(case['dim'])
                w = torch.softmax(s, -1)
                v = _wide(st, pages, slots, 1).transpose(0, 1).repeat_interleave(group, 0)
                out[b] = torch.matmul(w.contiguous(), v.contiguous()).transpose(0, 1)
            return out
        # many users: all positions at once, each user's sums by index
        user = torch.repeat_interleave(torch.arange(case['users']), torch.tensor(st['lens'])).to('cuda')
        first = torch.cumsum(torch.tensor([0] + st['lens']), 0)[:-1].to('cuda')
        pos = torch.arange(user.numel(), device='cuda') - first[user]
        for lo in range(0, case['users'], 512):
            mine = (user >= lo) & (user < lo + 512)
            u, p = user[mine], pos[mine]
            if not u.numel():
                continue
            pages, slots = st['table'].long()[u, p // case['page']], p % case['page']
            k, v = _wide(st, pages, slots, 0), _wide(st, pages, slots, 1)
            for h in range(case['q_heads']):
                for c in range(case['queries']):
                    s = (q[u, c, h] * k[:, h // group]).sum(-1) / math.sqrt(case['dim'])
                    top = torch.full((512,), -math.inf, dtype=torch.float64, device='cuda')
                    top = top.scatter_reduce(0, u - lo, s, 'amax')
                    w = torch.exp(s - top[u - lo])
                    total = torch.zeros(512, dtype=torch.float64, device='cuda').index_add(0, u - lo, w)
                    part = torch.zeros((512, case['dim']), dtype=torch.float64, device='cuda')
                    part = part.index_add(0, u - lo, w[:, None] * v[:, h // group])
                    part = part / torch.where(total > 0, total, torch.ones_like(total))[:, None]
                    out[lo:lo + 512, c, h] = part[:min(512, case['users'] - lo)]
        return out
    spots = [torch.arange(n - r, n) for n, r in zip(st['lens'], st['rows'])]
    pages = torch.cat([st['host_table'][b][s // case['page']] for b, s in enumerate(spots)]).long().to('cuda')
    slots = (torch.cat(spots) % case['page']).to('cuda')
    if case['op'] == 'read':
        return _wide(st, pages, slots, 0), _wide(st, pages, slots, 1)
    k, v = st['k'].double(), st['v'].double()
    if case['cache'] == 'e4m3':
        return _wide_quantised(k), _wide_quantised(v)
    pool = st['kv'].double()
    pool[pages, :, 0, slots] = k
    pool[pages, :, 1, slots] = v
    return pool
