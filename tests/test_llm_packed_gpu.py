"""GPU tests of the language-model operators for prompts laid end to end and for decode steps that share a prefix (packed.hip,
verify.hip), through ops.*, against plain implementations in 64 bits.

Attention tolerance, element by element.  With A = sum_j p_j |v_j| (64 bits): the probabilities are rounded to bf16 for the second
product (each off by at most 2^-8 of itself: 2^-8 A) and the result to bf16 (2^-8 |o|); scores are f32 sums of head_dim products, off by
at most (head_dim + 2) 2^-24 sum_d |q k| scale = delta, which moves a normalised probability by a factor within 1 +- 2 delta to first
order, the exponential adds 2^-21 (one unit of its f32 result, and the f32 rounding of its argument, of size up to 2^5, counted in
delta by two more products), and the sums over n keys at most n 2^-24 A each (numerator and denominator).
"""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, F64, I32 = torch.bfloat16, torch.float64, torch.int32


@pytest.fixture(scope='module')
def dev():
    from infernos_amd import _lib
    return _lib.require_device('cuda:0')


def i32(v, dev):
    return torch.tensor(v, dtype=I32, device=dev)


def attend64(q, k, v, scale):
    """one query head: q [d], k, v [n, d] -> (result, tolerance), 64 bits"""
    if k.size(0) == 0:
        z = torch.zeros_like(q)
        return z, z
    q, k, v = q.double(), k.double(), v.double()
    p = torch.softmax((k @ q) * scale, 0)
    o, A = p @ v, p @ v.abs()
    hd, n = q.numel(), k.size(0)
    delta = (hd + 4) * 2.0 ** -24 * float((k.abs() @ q.abs()).max()) * scale
    return o, 2.0 ** -8 * (A + o.abs()) + (2 * delta + 2.0 ** -20 + 2 * n * 2.0 ** -24) * A * 1.01 + 1e-30


def check_rows(out, rows, what):
    """rows: (index into out [N, nh, hd], o, tol)"""
    assert torch.isfinite(out).all(), what
    worst = 0.0
    for at, o, tol in rows:
        d = (out[at].double() - o).abs()
        assert bool((d <= tol).all()), (what, at, float(d.max()), float((d / tol.clamp(min=1e-30)).max()))
        worst = max(worst, float((d / tol.clamp(min=1e-30)).max()))
    return worst


def packed_case(dev, heads, lens, key_len, spare=0, extra_tokens=0, seed=0, max_keys=None):
    nh, nkv, hd = heads
    g = torch.Generator(device=dev).manual_seed(seed)
    N, n = sum(lens), len(lens)
    S = max(max(key_len), 1) + spare
    qkv = torch.randn(N + extra_tokens, (nh + 2 * nkv) * hd, generator=g, device=dev)
    qkv[:, :nh * hd] *= 2.0
    qkv = qkv.to(BF)
    cache = torch.randn(n, S, 2 * nkv * hd, generator=g, device=dev).to(BF)
    for s in range(n):
        cache[s, key_len[s]:] = float('nan')                        # slots behind key_len are not used
    cu = [0]
    for a in lens:
        cu.append(cu[-1] + a)
    return dict(heads=heads, lens=lens, cu=i32(cu, dev), key_len=i32(key_len, dev), klen=key_len, qkv=qkv, cache=cache, S=S, n=n, N=N + extra_tokens,
                max_keys=max(max(key_len), 1) if max_keys is None else max_keys)


def run_packed(c, dev, split=True, out=None):
    from infernos_amd import ops
    nh, nkv, hd = c['heads']
    kw = dict(ntokens=c['N'], nseqs=c['n'], nheads=nh, nkv=nkv, head_dim=hd, max_keys=c['max_keys'])
    ws = ops.attn_packed_ws(dev, **kw) if split else None
    if ws is not None:
        ws.fill_(float('nan'))
    if out is None:
        out = torch.full((c['N'], nh * hd), 7.0, dtype=BF, device=dev)
    ops.attn_packed(c['qkv'], c['cache'], out, c['cu'], c['key_len'], max_pos=c['S'], ws=ws, **kw)
    return out, ws


def packed_rows(c, sample=None):
    nh, nkv, hd = c['heads']
    G, i = nh // nkv, 0
    gen = torch.Generator().manual_seed(5)
    for s, n in enumerate(c['lens']):
        ts = range(n) if sample is None or n <= sample else sorted({0, n - 1, *torch.randint(0, n, (sample,), generator=gen).tolist()})
        for t in ts:
            m = max(0, min(c['klen'][s] - (n - 1 - t), c['klen'][s]))
            kv = c['cache'][s, :m].view(m, 2, nkv, hd)
            for h in range(nh) if sample is None else {0, nh - 1, (7 * t) % nh}:
                o, tol = attend64(c['qkv'][i + t, h * hd:(h + 1) * hd], kv[:, 0, h // G], kv[:, 1, h // G], hd ** -0.5)
                yield (i + t, h), o, tol
        i += n


HEADS = [(4, 1, 64), (2, 2, 128), (12, 2, 128), (14, 2, 64), (5, 1, 128), (16, 1, 64)]


@pytest.mark.parametrize('heads', HEADS)
@pytest.mark.parametrize('lens,past', [([1], 0), ([3, 1, 2], 0), ([5, 0, 33, 0], 0), ([64, 7], 0), ([21, 1, 4], 70), ([66], 130)])
def test_attn_packed_small(dev, heads, lens, past):
    """ragged sequences, empty ones among them, first prompts and later turns; every token and head"""
    c = packed_case(dev, heads, lens, [n + (past and past + 3 * s) for s, n in enumerate(lens)], spare=5, seed=len(lens) + past)
    nh, _, hd = heads
    out, _ = run_packed(c, dev)
    w = check_rows(out.view(-1, nh, hd), packed_rows(c), 'packed')
    print('attn_packed ok', heads, lens, past, 'worst share of the tolerance %.2f' % w)


@pytest.mark.parametrize('heads,lens,past', [((12, 2, 128), [700, 1, 65, 129, 640], 0), ((40, 8, 128), [257, 33], 1000), ((14, 2, 64), [1025], 0),
                                             ((4, 1, 64), [16], 5000), ((12, 2, 128), [1], 4095), ((16, 1, 128), [130], 900)])
def test_attn_packed_long(dev, heads, lens, past):
    """lengths past every tile and block edge, keys split over workgroups and not: the split changes no more than the roundings"""
    c = packed_case(dev, heads, lens, [n + (past + 11 * s if past else 0) for s, n in enumerate(lens)], spare=3, seed=9)
    nh, _, hd = heads
    rows = list(packed_rows(c, sample=12))
    for split in (False, True):
        out, ws = run_packed(c, dev, split)
        w = check_rows(out.view(-1, nh, hd), rows, 'packed split=%s' % split)
        print('attn_packed ok', heads, lens, past, 'split', ws is not None and ws.numel() > 0, 'worst share %.2f' % w)


@pytest.mark.parametrize('share', [0.9, 0.5, 0.26, 0.1, 0.0])
def test_smaller_workspaces_split_less(dev, share):
    """a workspace made for another batch: as many parts as it holds, the same results within the roundings"""
    heads = (12, 2, 128)
    c = packed_case(dev, heads, [20, 3], [3000, 1500], seed=12)
    full = run_packed(c, dev)[1]
    assert full.numel() > 0
    from infernos_amd import ops
    out = torch.empty(23, 12 * 128, dtype=BF, device=dev)
    n = int(full.numel() * share)
    guard = torch.full((n + 256,), 3.0, device=dev)
    ops.attn_packed(c['qkv'], c['cache'], out, c['cu'], c['key_len'], ntokens=23, nseqs=2, nheads=12, nkv=2, head_dim=128, max_pos=c['S'],
                    max_keys=c['max_keys'], ws=guard[:n])
    check_rows(out.view(-1, 12, 128), packed_rows(c, sample=4), 'packed')
    assert bool((guard[n:] == 3.0).all())
    x = prefix_case(dev, heads, 5, 2, 1500, [700, 20, 0, 300, 90], seed=13)
    kw = dict(nrows=5, tokens_per_row=2, prefix_keys=1500, nheads=12, nkv=2, head_dim=128, max_keys=x['max_keys'])
    full = ops.attn_prefix_ws(dev, **kw)
    two = 2 * 2 * 2 * 32 * 130                                       # parts x kv heads x row tiles x rows x (head_dim + 2)
    assert full.numel() > two
    n = max(two, int(full.numel() * share))
    guard = torch.full((n + 256,), 3.0, device=dev)
    check_rows(run_prefix(x, dev, ws=guard[:n]).view(-1, 12, 128), prefix_rows(x), 'prefix')
    assert bool((guard[n:] == 3.0).all())


def test_attn_packed_rows_that_see_nothing_and_tokens_behind_the_last(dev):
    """fewer keys than tokens: the first tokens see none and get zeros; tokens behind the last sequence keep what was there"""
    heads = (12, 2, 128)
    c = packed_case(dev, heads, [9, 70, 3], [4, 33, 0], spare=2, extra_tokens=6, seed=3)
    for split in (False, True):
        out, _ = run_packed(c, dev, split)
        o = out.view(-1, 12, 128)
        check_rows(o[:82], packed_rows(c), 'nothing')
        assert float(o[:5].abs().max()) == 0.0 and float(o[9:9 + 37].abs().max()) == 0.0 and float(o[79:82].abs().max()) == 0.0
        assert bool((o[82:] == 7.0).all())


@pytest.mark.parametrize('heads,lens,key_len', [((12, 2, 128), [40, 0, 33, 1, 64, 9], [5000, 300, 4000, 2000, 64, 0]),
                                                ((4, 1, 64), [40, 0, 33, 1, 64, 9], [5000, 300, 4000, 2000, 64, 0]),
                                                ((12, 2, 128), [2, 1, 0, 1, 1], [3001, 10, 700, 0, 1500]),
                                                ((4, 1, 64), [1, 0, 2] * 30, [700 - 7 * s for s in range(90)]),
                                                ((4, 1, 64), [1] * 200, [(37 * s) % 1200 for s in range(200)]),
                                                ((4, 1, 64), [1, 0, 2] * 30, [2600 - 29 * s for s in range(90)]),
                                                ((4, 1, 64), [1] * 200, [(137 * s) % 5000 for s in range(200)])])
def test_attn_packed_splits_ragged_sequences(dev, heads, lens, key_len):
    """few rows, long keys: sequences of every length share the workgroups, empty ones among them; tokens behind the last sequence keep
    what was there; without a workspace the same within the roundings"""
    c = packed_case(dev, heads, lens, key_len, spare=2, extra_tokens=40, seed=len(lens))
    nh, _, hd = heads
    N = sum(lens)
    rows = list(packed_rows(c, sample=6))
    out, ws = run_packed(c, dev)
    assert ws.numel() > 0 or max(key_len) <= 1200                     # (many short sequences fill the device whole)
    check_rows(out.view(-1, nh, hd), rows, 'split')
    assert bool((out[N:] == 7.0).all())
    out, _ = run_packed(c, dev, False)
    check_rows(out.view(-1, nh, hd), rows, 'whole')
    assert bool((out[N:] == 7.0).all())


def test_attn_packed_peaked_and_far_scores(dev):
    """scores spread over hundreds (one key takes it all), and all of one value"""
    heads = (4, 2, 128)
    c = packed_case(dev, heads, [70], [200], seed=4)
    c['qkv'][:, :512] *= 16.0
    out, _ = run_packed(c, dev)
    check_rows(out.view(-1, 4, 128), packed_rows(c, 8), 'peaked')
    c['qkv'][:, :512] = 0.0
    out, _ = run_packed(c, dev)
    check_rows(out.view(-1, 4, 128), packed_rows(c, 8), 'flat')


def test_attn_packed_masks_nan_and_inf_keys(dev):
    """a key that is NaN or infinite reaches only the tokens that see it (their values finite)"""
    heads = (4, 2, 128)
    c = packed_case(dev, heads, [80], [80], seed=6)
    c['cache'][0, 50, :128] = float('nan')
    c['cache'][0, 60, 128:256] = float('inf')
    out, _ = run_packed(c, dev, False)
    o = out.view(-1, 4, 128)
    check_rows(o[:50], (r for r in packed_rows(c) if r[0][0] < 50), 'masked')
    assert torch.isnan(o[50:, :2]).all() and torch.isfinite(o[50:60, 2:]).all()


def test_attn_packed_wrong_device_lengths_stay_in_range(dev):
    """offsets and lengths on the device that the host sizes do not allow are clamped"""
    heads = (4, 1, 64)
    c = packed_case(dev, heads, [8, 8], [30, 40], seed=7)
    ref, _ = run_packed(c, dev)
    ref = ref.clone()
    c['key_len'] = i32([30, 4000], dev)                               # past max_keys (40)
    out, _ = run_packed(c, dev)
    assert torch.equal(out, ref)
    c['cu'], c['key_len'] = i32([0, 8, 9000], dev), i32([30, -5], dev)
    out, _ = run_packed(c, dev)
    assert torch.equal(out[:8], ref[:8]) and float(out[8:].abs().max()) == 0.0


def prefix_case(dev, heads, B, T, P, own, plen=None, spare=4, seed=0):
    nh, nkv, hd = heads
    g = torch.Generator(device=dev).manual_seed(seed)
    S = max(own) + T + spare
    qkv = torch.randn(B * T, (nh + 2 * nkv) * hd, generator=g, device=dev)
    qkv[:, :nh * hd] *= 2.0
    key_len = [max(0, o + (t + 1 if o >= 0 else 0)) for o in own for t in range(T)]
    cache = torch.randn(B, S, 2 * nkv * hd, generator=g, device=dev).to(BF)
    for b in range(B):
        cache[b, key_len[b * T + T - 1]:] = float('nan')
    return dict(heads=heads, B=B, T=T, P=P, S=S, qkv=qkv.to(BF), cache=cache, prefix=torch.randn(P, 2 * nkv * hd, generator=g, device=dev).to(BF),
                klen=key_len, key_len=i32(key_len, dev), plen=plen, prefix_len=None if plen is None else i32(plen, dev),
                max_keys=max(1, max(key_len)))


def run_prefix(c, dev, out=None, ws=None):
    from infernos_amd import ops
    nh, nkv, hd = c['heads']
    kw = dict(nrows=c['B'], tokens_per_row=c['T'], prefix_keys=c['P'], nheads=nh, nkv=nkv, head_dim=hd, max_keys=c['max_keys'])
    if ws is None:
        ws = ops.attn_prefix_ws(dev, **kw).fill_(float('nan'))
    if out is None:
        out = torch.full((c['B'] * c['T'], nh * hd), 7.0, dtype=BF, device=dev)
    ops.attn_prefix(c['qkv'], c['prefix'], c['cache'], out, c['key_len'], max_pos=c['S'], prefix_len=c['prefix_len'], ws=ws, **kw)
    return out


def prefix_rows(c, sample=None):
    nh, nkv, hd = c['heads']
    G = nh // nkv
    for i in range(c['B'] * c['T']):
        b, m = i // c['T'], c['klen'][i]
        x = c['P'] if c['plen'] is None else c['plen'][b]
        kv = torch.cat([c['prefix'][:x], c['cache'][b, :m]]).view(x + m, 2, nkv, hd)
        if sample is not None and i % sample:
            continue
        for h in range(nh) if sample is None else {i % nh, nh - 1}:
            o, tol = attend64(c['qkv'][i, h * hd:(h + 1) * hd], kv[:, 0, h // G], kv[:, 1, h // G], hd ** -0.5)
            yield (i, h), o, tol


@pytest.mark.parametrize('heads', HEADS)
@pytest.mark.parametrize('B,T,P', [(1, 1, 1), (3, 1, 63), (2, 4, 65), (5, 3, 300)])
def test_attn_prefix_small(dev, heads, B, T, P):
    c = prefix_case(dev, heads, B, T, P, [(17 * b) % 90 for b in range(B)], seed=B + P)
    w = check_rows(run_prefix(c, dev).view(-1, heads[0], heads[2]), prefix_rows(c), 'prefix')
    print('attn_prefix ok', heads, B, T, P, 'worst share %.2f' % w)


@pytest.mark.parametrize('heads,B,T,P,own', [((12, 2, 128), 64, 1, 2048, 300), ((40, 8, 128), 9, 5, 1501, 700), ((14, 2, 64), 33, 2, 777, 40),
                                             ((12, 2, 128), 1, 1, 6000, 2100), ((4, 1, 64), 96, 6, 129, 10)])
def test_attn_prefix_batches(dev, heads, B, T, P, own):
    """decode batches and drafted tokens; rows that use all, a part or none of the prefix"""
    plen = [P if b % 3 else (P * b // max(1, B)) for b in range(B)]
    c = prefix_case(dev, heads, B, T, P, [(own * (b + 1) * 7919 % (own + 1)) for b in range(B)], plen=plen, seed=P)
    w = check_rows(run_prefix(c, dev).view(-1, heads[0], heads[2]), prefix_rows(c, sample=max(1, B * T // 24)), 'prefix')
    print('attn_prefix ok', heads, B, T, P, own, 'worst share %.2f' % w)


@pytest.mark.parametrize('heads,B,T,P,own', [((40, 8, 128), 64, 5, 1000, 300), ((8, 8, 64), 96, 6, 700, 90), ((16, 1, 128), 96, 6, 3000, 500),
                                             ((14, 2, 64), 90, 6, 2500, 33), ((40, 8, 128), 40, 7, 97, 2000)])
def test_attn_prefix_both_key_sets_fill_the_device(dev, heads, B, T, P, own):
    """hundreds of workgroups of either key set; rows without an own key and rows that use none of the prefix among them"""
    plen = [0 if b % 11 == 3 else P if b % 4 else 1 + (P * 7 * b) % P for b in range(B)]
    c = prefix_case(dev, heads, B, T, P, [-1 if b % 13 == 5 else (b * 7919) % (own + 1) for b in range(B)], plen=plen, seed=own)
    w = check_rows(run_prefix(c, dev).view(-1, heads[0], heads[2]), prefix_rows(c, sample=7), 'prefix')
    print('attn_prefix ok', heads, B, T, P, own, 'worst share %.2f' % w)


def test_attn_prefix_rows_that_see_nothing(dev):
    """no prefix and no key: zeros; no prefix, or no own key: the other alone"""
    heads = (12, 2, 128)
    c = prefix_case(dev, heads, 4, 1, 200, [-1, 20, -1, 70], plen=[0, 0, 200, 130], seed=2)
    out = run_prefix(c, dev).view(4, 12, 128)
    check_rows(out, prefix_rows(c), 'none')
    assert float(out[0].abs().max()) == 0.0
    c['prefix_len'], c['key_len'] = i32([-3, 1 << 30, 200, 130], dev), i32([-9, 1 << 30, 0, 71], dev)      # clamped to the host sizes
    c['cache'] = torch.nan_to_num(c['cache'], nan=0.5)
    c['plen'], c['klen'] = [0, 200, 200, 130], [0, c['max_keys'], 0, 71]
    check_rows(run_prefix(c, dev).view(4, 12, 128), prefix_rows(c), 'clamped')


def test_attention_offsets_past_32_bits(dev):
    """a cache row whose keys lie more than 2^32 bytes apart, and a second row 2^31 elements behind the first"""
    from infernos_amd import ops
    nh, nkv, hd, K = 8, 8, 128, (1 << 20) + 70000
    ts = 2 * nkv * hd                                                # 4 KB a slot: 2^20 slots = 4 GiB
    g = torch.Generator(device=dev).manual_seed(1)
    cache = torch.empty(2, K, ts, dtype=BF, device=dev)
    for b in range(2):
        for a in range(0, K, 1 << 17):
            cache[b, a:a + (1 << 17)].normal_(generator=g)
    q = torch.randn(2, nh * hd, generator=g, device=dev).to(BF) * 2
    q[:, -hd:] *= 4
    lens = [K, K - 33]
    out = torch.empty(2, nh * hd, dtype=BF, device=dev)
    kw = dict(ntokens=2, nseqs=2, nheads=nh, nkv=nkv, head_dim=hd, max_keys=K)
    ops.attn_packed(q, cache, out, i32([0, 1, 2], dev), i32(lens, dev), max_pos=K, q_ts=nh * hd, ws=ops.attn_packed_ws(dev, **kw), **kw)
    pre = torch.empty_like(out)
    pk = dict(nrows=2, tokens_per_row=1, prefix_keys=K, nheads=nh, nkv=nkv, head_dim=hd, max_keys=K)
    ops.attn_prefix(q, cache[1], cache, pre, i32([0, lens[1]], dev), max_pos=K, q_ts=nh * hd, prefix_len=i32([lens[1], 0], dev),
                    ws=ops.attn_prefix_ws(dev, **pk), **pk)
    for h in (0, 7):
        sl = slice(h * hd, (h + 1) * hd)
        ref = [attend64(q[b, sl], cache[b, :lens[b], sl], cache[b, :lens[b], nkv * hd + h * hd:nkv * hd + (h + 1) * hd], hd ** -0.5) for b in range(2)]
        cross = attend64(q[0, sl], cache[1, :lens[1], sl], cache[1, :lens[1], nkv * hd + h * hd:nkv * hd + (h + 1) * hd], hd ** -0.5)
        for got, (o, tol) in ((out[0], ref[0]), (out[1], ref[1]), (pre[0], cross), (pre[1], ref[1])):
            assert bool(((got[sl].double() - o).abs() <= tol).all())


@pytest.mark.parametrize('heads', [(4, 1, 64), (12, 2, 128), (5, 5, 128)])
def test_rope_append_packed(dev, heads):
    """the bits of ops.rope_append on the same tokens padded; slots apart from positions; q in place or apart; nothing else written"""
    from infernos_amd import ops
    nh, nkv, hd = heads
    g = torch.Generator(device=dev).manual_seed(nh)
    lens, past, S = [5, 0, 1, 17], [0, 3, 40, 7], 64
    N, T, n = sum(lens), max(lens), len(lens)
    W = (nh + 2 * nkv) * hd
    ang = torch.arange(S, device=dev, dtype=F64)[:, None] * 1.0e4 ** (-torch.arange(0, hd, 2, device=dev, dtype=F64) / hd)
    cs = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    qkv = torch.randn(N + 2, W, generator=g, device=dev).to(BF)
    cache0 = torch.randn(n, S, 2 * nkv * hd, generator=g, device=dev).to(BF)
    cu = [0]
    for a in lens:
        cu.append(cu[-1] + a)
    pad = torch.zeros(n, T, W, dtype=BF, device=dev)
    for s, a in enumerate(lens):
        pad[s, :a] = qkv[cu[s]:cu[s + 1]]
    ref_cache = cache0.clone()
    ops.rope_append(pad, cs, ref_cache, i32(past, dev), i32(lens, dev), nrows=n, tokens_per_row=T, nheads=nh, nkv=nkv, head_dim=hd, max_pos=S)
    kw = dict(ntokens=N + 2, nseqs=n, nheads=nh, nkv=nkv, head_dim=hd, max_pos=S)
    cache, q = cache0.clone(), torch.full((N + 2, nh * hd), 7.0, dtype=BF, device=dev)
    src = qkv.clone()
    ops.rope_append_packed(src, cs, cache, i32(cu, dev), i32(past, dev), q_out=q, **kw)
    assert torch.equal(src, qkv) and torch.equal(cache, ref_cache)
    for s, a in enumerate(lens):
        assert torch.equal(q[cu[s]:cu[s + 1]], pad[s, :a, :nh * hd])
    assert bool((q[N:] == 7.0).all())
    cache = cache0.clone()
    ops.rope_append_packed(src, cs, cache, i32(cu, dev), i32(past, dev), **kw)
    assert torch.equal(src[:N, :nh * hd], q[:N]) and torch.equal(src[:, nh * hd:], qkv[:, nh * hd:]) and torch.equal(src[N:], qkv[N:])
    # slots apart from positions; against the formula in 64 bits: products and their sum in f32, one rounding to bf16
    cache, slot0 = cache0.clone(), [10, 0, 63, 60]
    ops.rope_append_packed(qkv.clone(), cs, cache, i32(cu, dev), i32(past, dev), slot0=i32(slot0, dev), **kw)
    want, tol = cache0.double(), torch.zeros(cache0.shape, dtype=F64, device=dev)
    for s, a in enumerate(lens):
        for t in range(a):
            if slot0[s] + t >= S:
                continue                                             # outside the row: left alone
            x = qkv[cu[s] + t].double().view(-1, hd)
            c, sn = cs[past[s] + t].double().unbind(-1)
            lo, hi = x[nh:nh + nkv, :hd // 2], x[nh:nh + nkv, hd // 2:]
            want[s, slot0[s] + t, :nkv * hd] = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1).reshape(-1)
            mag = torch.cat([(lo * c).abs() + (hi * sn).abs(), (hi * c).abs() + (lo * sn).abs()], -1).reshape(-1)
            tol[s, slot0[s] + t, :nkv * hd] = 2.0 ** -8 * want[s, slot0[s] + t, :nkv * hd].abs() + 1.01 * 2.0 ** -23 * mag
            want[s, slot0[s] + t, nkv * hd:] = x[nh + nkv:].reshape(-1)
    assert bool(((cache.double() - want).abs() <= tol).all())
    # positions outside the table: left alone
    cache, q = cache0.clone(), torch.full((N + 2, nh * hd), 7.0, dtype=BF, device=dev)
    ops.rope_append_packed(qkv.clone(), cs, cache, i32(cu, dev), i32([-5, 0, S, S - 1], dev), slot0=i32([0, 0, 0, 0], dev), q_out=q, **kw)
    assert torch.equal(cache[2], cache0[2]) and torch.equal(cache[0], cache0[0]) and not torch.equal(cache[3, 0], cache0[3, 0])
    assert torch.equal(cache[3, 1:], cache0[3, 1:]) and bool((q[:6] == 7.0).all())


@pytest.mark.parametrize('n', [65, 300, 5000])
def test_many_sequences_most_of_them_empty(dev, n):
    """hundreds and thousands of sequences, one token or none each: every one found (rows and positions by their number)"""
    from infernos_amd import ops
    nh, nkv, hd = 4, 1, 64
    g = torch.Generator(device=dev).manual_seed(n)
    lens = [(1 if (s * 7919) % 5 == 0 else 0) + (3 if s % 97 == 5 else 0) for s in range(n)]
    N = sum(lens)
    key_len = [a + s % 3 for s, a in enumerate(lens)]
    c = packed_case(dev, (nh, nkv, hd), lens, key_len, seed=n)
    out, _ = run_packed(c, dev)
    for (i, h), o, t in packed_rows(c, sample=2 if n > 1000 else None):
        assert bool(((out.view(N, nh, hd)[i, h].double() - o).abs() <= t).all()), (i, h)
    ang = torch.arange(16, device=dev, dtype=F64)[:, None] * 1.0e4 ** (-torch.arange(0, hd, 2, device=dev, dtype=F64) / hd)
    cs = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    cache = torch.zeros(n, 8, 2 * nkv * hd, dtype=BF, device=dev)
    pos0 = [s % 4 for s in range(n)]
    ops.rope_append_packed(c['qkv'], cs, cache, c['cu'], i32(pos0, dev), ntokens=N, nseqs=n, nheads=nh, nkv=nkv, head_dim=hd, max_pos=8)
    ref, i = torch.zeros_like(cache), 0
    for s, a in enumerate(lens):
        ref[s, pos0[s]:pos0[s] + a, hd:] = c['qkv'][i:i + a, (nh + 1) * hd:]
        i += a
    assert torch.equal(cache[:, :, hd:], ref[:, :, hd:])


# ---- drafts -------------------------------------------------------------------------------------------------------------
def verify64(p, q, drafts, u, n):
    """p [n + 1, V], q [n, V] f64 rows of one request -> (kept, mass of the drawn position, margin of the closest decision)"""
    margin = 1.0
    for i in range(n):
        x = int(drafts[i])
        px, qx = (float(p[i, x]), float(q[i, x])) if 0 <= x < p.size(1) else (0.0, 1.0)
        margin = min(margin, abs(float(u[i]) * qx - px)) if px or qx else margin
        if not float(u[i]) * qx < px:
            rest = (p[i] - q[i]).clamp(min=0)
            return i, (rest if float(rest.sum()) > 0 else p[i]), margin
    return n, p[n], margin


def check_verified(tokens, count, r, kept, mass, drafts, u_draw, order=None):
    """the drawn token's interval of the cumulated mass holds the uniform number.  Exponentials are good to 1e-10 of themselves and the
    sum they are divided by to as much, so that any sum of p is within 2e-10 (p sums to 1), on both sides of the comparison: 4e-10, and
    f64 sums of 2e5 terms, 2e5 2^-53 < 1e-10 of the whole"""
    T1 = tokens.size(1)
    assert int(count[r]) == kept + 1, (r, int(count[r]), kept)
    assert tokens[r, :kept].tolist() == [int(x) for x in drafts[:kept]]
    assert tokens[r, kept + 1:].tolist() == [-1] * (T1 - kept - 1)
    tok = int(tokens[r, kept])
    if float(mass.sum()) == 0.0:
        assert tok == -1
        return
    at = tok if order is None else order.index(tok)
    c = mass.cumsum(0)
    tot, hi = float(c[-1]), float(c[at])
    lo, off = hi - float(mass[at]), 4e-10 + 1e-10 * tot
    assert float(mass[at]) > 0 and lo <= u_draw * tot + off and hi > u_draw * tot - off, (r, tok, lo, hi, u_draw * tot)


def run_verify(dev, logits, drafts, u, V, temperature, q=None, lens=None, ld=None):
    from infernos_amd import ops
    B, T1 = u.shape
    tok, cnt = torch.full((B, T1), -7, dtype=I32, device=dev), torch.full((B,), -7, dtype=I32, device=dev)
    ws = ops.verify_drafts_ws(B, T1 - 1, dev)
    ws.fill_(255)
    ops.verify_drafts(logits, drafts, u, tok, cnt, ws, vocab=V, ld=logits.size(-1) if ld is None else ld, nrows=B, ndraft=T1 - 1,
                      temperature=temperature, draft_probs=q, lens=lens, q_ld=None if q is None else q.size(-1))
    return tok.cpu(), cnt.cpu()


@pytest.mark.parametrize('B,T,V,temp,probs,pad', [(1, 1, 5, 1.0, True, 0), (7, 4, 777, 0.7, True, 3), (9, 3, 8192, 1.0, False, 0), (5, 6, 8193, 1.3, True, 3),
                                                  (6, 2, 151936, 0.8, True, 0), (3, 3, 152064, 1.0, False, 1), (4, 0, 1000, 1.0, False, 0), (2, 63, 33, 0.9, True, 0)])
def test_verify_drafts(dev, B, T, V, temp, probs, pad):
    """whole distributions; odd vocabularies and strides, rows of their own draft counts"""
    g = torch.Generator(device=dev).manual_seed(V + B)
    logits = torch.randn(B * (T + 1), V + pad, generator=g, device=dev) * 2
    logits[:, :5] += 6
    lv = logits[:, :V].double() / temp
    p = torch.softmax(lv, -1).view(B, T + 1, V)
    q = None
    if T:
        d = logits.view(B, T + 1, V + pad)[:, :T] + 0.5 * torch.randn(B, T, V + pad, generator=g, device=dev)
        q = torch.softmax(d[..., :V] / temp, -1).reshape(B * T, V)
        drafts = torch.multinomial(q, 1, generator=g).view(B, T).to(I32)
        q = torch.nn.functional.pad(q, (0, pad), value=0.5).contiguous()
    else:
        drafts = torch.zeros(B, 1, dtype=I32, device=dev)
    u = torch.rand(B, T + 1, generator=g, device=dev)
    lens = None if B % 2 else [min(T, r % (T + 1) + (r == 0)) for r in range(B)]
    tok, cnt = run_verify(dev, logits, drafts, u, V, temp, q if probs and T else None, None if lens is None else i32(lens, dev))
    seen = set()
    for r in range(B):
        n = T if lens is None else lens[r]
        qr = q[r * T:(r + 1) * T, :V].double() if probs and T else torch.nn.functional.one_hot(drafts[r].long()[:T], V).double() if T else None
        kept, mass, margin = verify64(p[r], qr, drafts[r], u[r], n)
        assert margin > 1e-10
        check_verified(tok, cnt, r, kept, mass, drafts[r].cpu(), float(u[r, T]))
        seen.add(kept)
    print('verify ok', B, T, V, 'kept', sorted(seen))


def test_verify_drafts_greedy_ties_and_masks(dev):
    """temperature 0 (lowest id of equals), -inf and NaN logits, rows with nothing left, drafts outside the vocabulary, q above p everywhere
    it matters, uniform numbers at the ends"""
    V = 9000
    inf = float('inf')
    l = torch.full((2 * 3, V), -1.0, device=dev)
    l[0, 8500] = l[0, 100] = 4.0
    l[1, 7] = 9.0
    l[2, 8999] = 2.0
    l[3] = -inf
    l[4, 1] = l[5, 2] = 1.0
    drafts = i32([[100, 7], [3, 1]], dev)
    u = torch.full((2, 3), 0.999, device=dev)
    tok, cnt = run_verify(dev, l, drafts, u, V, 0.0)
    assert tok.tolist() == [[100, 7, 8999], [-1, -1, -1]] and cnt.tolist() == [3, 1]
    drafts[0, 0] = 8500                                              # equal, but not the lowest id
    tok, cnt = run_verify(dev, l, drafts, u, V, 0.0)
    assert tok[0].tolist() == [100, -1, -1] and int(cnt[0]) == 1
    # drawn: NaN and -inf are never chosen, +inf always; a draft out of range is refused, nothing read out of range
    l = torch.full((5 * 2, V), -inf, device=dev)
    l[0, 4000] = 0.0                                                 # one token left
    l[1, 0] = l[1, 8999] = 3.0
    l[2] = 0.0
    l[2, 17] = float('nan')
    l[3, 5] = inf
    l[4, 10] = l[4, 20] = l[5, 6] = 0.0
    l[6] = -inf
    l[7, 1] = 1.0
    l[8, 30] = l[8, 40] = l[9, 3] = 1.0
    drafts = i32([[4000], [17], [V], [0], [-1]], dev)
    u = torch.tensor([[0.5, 0.75], [0.0, 0.0], [0.0, 0.5], [0.0, 0.3], [0.0, 0.49]], device=dev)
    tok, cnt = run_verify(dev, l, drafts, u, V, 1.0)
    assert tok.tolist() == [[4000, 8999], [0, -1], [20, -1], [-1, -1], [30, -1]] and cnt.tolist() == [2, 1, 1, 1, 1]
    # p = q: every draft is kept; with the draft refused by q = 1 at a token p barely has, the rest is p elsewhere
    p = torch.softmax(torch.randn(2, V, device=dev), -1)
    l = torch.stack([p[0].log(), p[1].log()])
    tok, cnt = run_verify(dev, l, i32([[77]], dev), torch.tensor([[0.9990, 0.5]], device=dev), V, 1.0, q=p[:1].contiguous())
    assert int(cnt[0]) == 2 and int(tok[0, 0]) == 77
    tok, cnt = run_verify(dev, l, i32([[77]], dev), torch.tensor([[0.999, 0.0]], device=dev), V, 1.0)
    assert tok.tolist() == [[0, -1]]
    tok, cnt = run_verify(dev, l, i32([[0]], dev), torch.tensor([[0.999, 0.0]], device=dev), V, 1.0)
    assert tok.tolist() == [[1, -1]]
    # a number at or past 1 (a caller's rounding): the last token with any mass
    l2 = torch.full((1, V), -inf, device=dev)
    l2[0, 3], l2[0, 4000] = 1.0, 2.0
    tok, cnt = run_verify(dev, l2, i32([[0]], dev), torch.tensor([[1.0]], device=dev), V, 1.0)
    assert tok.tolist() == [[4000]] and cnt.tolist() == [1]
    # the draft's distribution covers the target's: nothing is left over, so the token comes from p
    big = torch.ones(1, V, device=dev)
    tok, cnt = run_verify(dev, l, i32([[77]], dev), torch.tensor([[0.999, 0.99999]], device=dev), V, 1.0, q=big)
    check_verified(tok, cnt, 0, 0, torch.softmax(l[0].double(), 0), [77], float(torch.tensor(0.99999)))


@pytest.mark.parametrize('B,T,probs', [(1, 1, True), (33, 4, True), (17, 3, False), (4, 0, False)])
def test_verify_drafts_topk_behind_the_sampler(dev, B, T, probs):
    """on what ops.sample_topk says of the target's and the draft's logits, drafts drawn by it"""
    from infernos_amd import ops
    V = 1000
    g = torch.Generator(device=dev).manual_seed(B)

    def dist(logits):
        n = logits.size(0)
        cand, pr = torch.zeros(n, 32, dtype=I32, device=dev), torch.zeros(n, 32, device=dev)
        tok = torch.zeros(n, dtype=I32, device=dev)
        ops.sample_topk(logits, torch.rand(n, generator=g, device=dev), tok, torch.zeros(n * 260, dtype=torch.uint8, device=dev), vocab=V, ld=V,
                        nrows=n, temperature=0.7, top_k=20, top_p=0.8, out_cand=cand, out_probs=pr)
        return tok, cand, pr

    target = torch.randn(B * (T + 1), V, generator=g, device=dev) * 1.5
    _, cand, pr = dist(target)
    drafts, dc, dp = torch.zeros(B, max(T, 1), dtype=I32, device=dev), None, None
    if T:
        near = (target.view(B, T + 1, V)[:, :T] + 0.3 * torch.randn(B, T, V, generator=g, device=dev)).reshape(B * T, V).contiguous()
        tok, dc, dp = dist(near)
        drafts = tok.view(B, T).contiguous()
    u = torch.rand(B, T + 1, generator=g, device=dev)
    lens = [T if r % 5 else T // 2 for r in range(B)]
    out, cnt = torch.full((B, T + 1), -7, dtype=I32, device=dev), torch.full((B,), -7, dtype=I32, device=dev)
    ops.verify_drafts_topk(cand, pr, drafts, u, out, cnt, nrows=B, ndraft=T, draft_cand=dc if probs else None,
                           draft_probs=dp if probs else None, lens=i32(lens, dev))
    out, cnt = out.cpu(), cnt.cpu()
    kepts = set()
    for r in range(B):
        def row(c, p):
            return torch.zeros(V, dtype=F64, device=dev).index_add_(0, c.long(), p.double())
        p = torch.stack([row(cand[r * (T + 1) + i], pr[r * (T + 1) + i]) for i in range(T + 1)])
        q = torch.stack([row(dc[r * T + i], dp[r * T + i]) if probs else torch.nn.functional.one_hot(drafts[r, i].long(), V).double()
                         for i in range(T)]) if T else None
        kept, mass, margin = verify64(p, q, drafts[r], u[r], lens[r])
        assert margin > 1e-10 or T == 0
        order = cand[r * (T + 1) + kept].tolist()
        check_verified(out, cnt, r, kept, mass[cand[r * (T + 1) + kept].long()], drafts[r].cpu(), float(u[r, T]), order)
        kepts.add(kept)
    print('verify topk ok', B, T, 'kept', sorted(kepts))


def test_verified_tokens_follow_the_targets_distribution(dev):
    """20 000 independent draws from a draft, verified: the first token's frequencies are the target's (five standard deviations)"""
    V, B = 12, 20000
    g = torch.Generator(device=dev).manual_seed(11)
    p, q = torch.softmax(torch.randn(V, generator=g, device=dev), 0), torch.softmax(torch.randn(V, generator=g, device=dev), 0)
    logits = p.log().expand(B, 2, V).reshape(B * 2, V).contiguous()
    drafts = torch.multinomial(q, B, replacement=True, generator=g).to(I32).view(B, 1)
    tok, _ = run_verify(dev, logits, drafts, torch.rand(B, 2, generator=g, device=dev), V, 1.0, q=q.expand(B, V).contiguous())
    f = torch.bincount(tok[:, 0].long(), minlength=V).double() / B
    pd = p.double().cpu()
    assert bool(((f - pd).abs() <= 5 * (pd * (1 - pd) / B).sqrt()).all()), (f, pd)


# ---- streams, graphs, together ----------------------------------------------------------------------------------------------
def test_other_stream_and_captured_graph_replays(dev):
    """one capture of the step's four operators on a side stream, replayed with new inputs and lengths, eager work between: every replay
    is the eager result bit for bit"""
    from infernos_amd import _lib, ops
    heads = nh, nkv, hd = (12, 2, 128)
    c = packed_case(dev, heads, [130, 1, 67], [2000, 1500, 1700], spare=8, seed=20)
    x = prefix_case(dev, heads, 6, 2, 900, [100, 5, 0, 33, 64, 80], seed=21)
    V, B, T = 9000, 6, 1
    logits, u = torch.randn(B * 2, V, device=dev), torch.rand(B, 2, device=dev)
    drafts = i32([[1], [2], [3], [4], [5], [6]], dev)
    pw = ops.attn_packed_ws(dev, ntokens=c['N'], nseqs=3, nheads=nh, nkv=nkv, head_dim=hd, max_keys=c['max_keys'])
    assert pw.numel() > 0
    xw = ops.attn_prefix_ws(dev, nrows=6, tokens_per_row=2, prefix_keys=900, nheads=nh, nkv=nkv, head_dim=hd, max_keys=x['max_keys'])
    vw = ops.verify_drafts_ws(B, T, dev)
    o1, o2 = torch.zeros(c['N'], nh * hd, dtype=BF, device=dev), torch.zeros(12, nh * hd, dtype=BF, device=dev)
    tok, cnt = torch.zeros(B, 2, dtype=I32, device=dev), torch.zeros(B, dtype=I32, device=dev)

    def step():
        ops.attn_packed(c['qkv'], c['cache'], o1, c['cu'], c['key_len'], ntokens=c['N'], nseqs=3, nheads=nh, nkv=nkv, head_dim=hd,
                        max_pos=c['S'], max_keys=c['max_keys'], ws=pw)
        run_prefix(x, dev, out=o2, ws=xw)
        ops.verify_drafts(logits, drafts, u, tok, cnt, vw, vocab=V, ld=V, nrows=B, ndraft=T)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = _lib.CountedGraph(step)
        for k in range(4):
            c['qkv'].add_(0.25)
            x['qkv'].mul_(0.9)
            logits.mul_(1.1)
            u.copy_(torch.rand(B, 2, device=dev))
            if k == 2:
                c['key_len'].copy_(i32([1990, 700, 1600], dev))
            step()
            want = [t.clone() for t in (o1, o2, tok, cnt)]
            for t in (o1, o2, tok, cnt):
                t.zero_()
            if k % 2:
                side.synchronize()
            graph.replay()
            for a, b in zip(want, (o1, o2, tok, cnt)):
                assert torch.equal(a, b), k
    torch.cuda.current_stream(dev).wait_stream(side)
    with torch.cuda.stream(side):
        pass


def test_two_streams_with_a_workspace_each(dev):
    """the same calls at once on two streams, each with its own workspace and output"""
    heads = (12, 2, 128)
    x = prefix_case(dev, heads, 8, 1, 3000, [60 * b for b in range(8)], seed=31)
    y = prefix_case(dev, heads, 8, 1, 3000, [50 * b for b in range(8)], seed=32)
    want = [run_prefix(x, dev).clone(), run_prefix(y, dev).clone()]
    torch.cuda.synchronize()
    from infernos_amd import ops
    ws = [ops.attn_prefix_ws(dev, nrows=8, tokens_per_row=1, prefix_keys=3000, nheads=12, nkv=2, head_dim=128, max_keys=z['max_keys']) for z in (x, y)]
    outs = [torch.zeros_like(w) for w in want]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(dev), torch.cuda.Stream(dev)]
    for _ in range(20):
        for s, z, o, w in zip(streams, (x, y), outs, ws):
            with torch.cuda.stream(s):
                run_prefix(z, dev, out=o, ws=w)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_a_drafted_step_behind_a_shared_prefix(dev):
    """the operators as a server uses them, one attention layer: the prefix appended and attended once as a packed prompt, the rows'
    prompts appended at slots of their own and attended behind it, then a step of three drafted tokens a row; each stage against 64 bits
    of what the stage before left in the cache"""
    from infernos_amd import ops
    nh, nkv, hd, S, P = 12, 2, 128, 96, 150
    G, W, KV = nh // nkv, (nh + 2 * nkv) * hd, 2 * nkv * hd
    g = torch.Generator(device=dev).manual_seed(40)
    new = lambda n: torch.randn(n, W, generator=g, device=dev).to(BF)
    ang = torch.arange(512, device=dev, dtype=F64)[:, None] * 1.0e6 ** (-torch.arange(0, hd, 2, device=dev, dtype=F64) / hd)
    cs = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    H = dict(nheads=nh, nkv=nkv, head_dim=hd)

    prefix = torch.zeros(1, P, KV, dtype=BF, device=dev)
    qkv = new(P)
    ops.rope_append_packed(qkv, cs, prefix, i32([0, P], dev), i32([0], dev), ntokens=P, nseqs=1, max_pos=P, **H)
    out = torch.empty(P, nh * hd, dtype=BF, device=dev)
    kw = dict(ntokens=P, nseqs=1, max_keys=P, **H)
    ops.attn_packed(qkv, prefix, out, i32([0, P], dev), i32([P], dev), max_pos=P, ws=ops.attn_packed_ws(dev, **kw), **kw)
    rows = []
    for t in (0, 77, P - 1):
        kv = prefix[0, :t + 1].view(-1, 2, nkv, hd)
        for h in (0, 11):
            rows.append(((t, h), *attend64(qkv[t, h * hd:(h + 1) * hd], kv[:, 0, h // G], kv[:, 1, h // G], hd ** -0.5)))
    check_rows(out.view(P, nh, hd), rows, 'prefix prompt')

    cache = torch.full((3, S, KV), float('nan'), dtype=BF, device=dev)
    have = [0, 0, 0]
    for lens in ([40, 1, 7], [3, 3, 3]):                              # the rows' own prompts, then three drafted tokens each
        T = max(lens)
        cu = [0, lens[0], lens[0] + lens[1], sum(lens)]
        qkv = new(sum(lens))
        ops.rope_append_packed(qkv, cs, cache, i32(cu, dev), i32([P + a for a in have], dev), slot0=i32(have, dev), ntokens=cu[3], nseqs=3, max_pos=S, **H)
        # padded to T tokens a row, as the decode step's buffers are; padding tokens see nothing of the row
        q = torch.zeros(3 * T, W, dtype=BF, device=dev)
        klen = [0] * (3 * T)
        for b in range(3):
            q[b * T:b * T + lens[b]] = qkv[cu[b]:cu[b + 1]]
            for t in range(lens[b]):
                klen[b * T + t] = have[b] + t + 1
        out = torch.empty(3 * T, nh * hd, dtype=BF, device=dev)
        kw = dict(nrows=3, tokens_per_row=T, prefix_keys=P, max_keys=S, **H)
        ops.attn_prefix(q, prefix, cache, out, i32(klen, dev), max_pos=S, ws=ops.attn_prefix_ws(dev, **kw), **kw)
        rows = []
        for i in range(3 * T):
            b, m = i // T, klen[i]
            if i % T >= lens[b]:
                continue
            kv = torch.cat([prefix[0], cache[b, :m]]).view(-1, 2, nkv, hd)
            for h in (i % nh, 5):
                rows.append(((i, h), *attend64(q[i, h * hd:(h + 1) * hd], kv[:, 0, h // G], kv[:, 1, h // G], hd ** -0.5)))
        check_rows(out.view(3 * T, nh, hd), rows, 'rows %s' % lens)
        have = [a + b for a, b in zip(have, lens)]

    # the drafted step's logits (here: a projection of the attention's result), verified
    V = 500
    logits = (out.float() @ torch.randn(nh * hd, V, generator=g, device=dev)).contiguous() * 0.05
    drafts = logits.view(3, 3, V)[:, :2].argmax(-1).to(I32).contiguous()
    u = torch.rand(3, 3, generator=g, device=dev)
    tok, cnt = run_verify(dev, logits, drafts, u, V, 0.7)
    p = torch.softmax(logits.double() / 0.7, -1).view(3, 3, V)
    for r in range(3):
        kept, mass, margin = verify64(p[r], torch.nn.functional.one_hot(drafts[r].long(), V).double(), drafts[r], u[r], 2)
        assert margin > 1e-10
        check_verified(tok, cnt, r, kept, mass, drafts[r].cpu(), float(u[r, 2]))
