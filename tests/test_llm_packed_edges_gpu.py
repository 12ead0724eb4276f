"""GPU tests of packed.hip and verify.hip where the first ones do not reach: the bits that the probabilities keep, scores that leave the
first tile empty, every kernel form, and draft verification at the sizes of a server's batch.  References in 64 bits."""
import pytest
import torch

from test_llm_packed_gpu import BF, F64, check_verified, dev, i32, packed_case, prefix_case, verify64        # noqa: F401  (dev is a fixture)

pytestmark = pytest.mark.gpu


def attend_f32(q, k, v, scale):
    """one query head -> (result in 64 bits, tolerance of a kernel whose probabilities keep 16 bits).  With A = sum_j p_j |v_j|: the
    result's rounding to bf16, 2^-8 |o|; a probability as the sum of two bf16, each off by at most 2^-8 of what it rounds: 2^-16 A; a
    score is an f32 sum of head_dim products, off by at most (head_dim + 4) 2^-24 sum_d |q k| scale = delta (the scaling and the
    exponent's argument are two roundings each), which moves a normalised probability by 2 delta; the exponential 2^-21 and the
    polynomial of its argument's range 2^-21 more; sums over n keys n 2^-24 A in numerator and denominator"""
    if k.size(0) == 0:
        z = torch.zeros_like(q, dtype=F64)
        return z, z
    q, k, v = q.double(), k.double(), v.double()
    p = torch.softmax((k @ q) * scale, 0)
    o, A = p @ v, p @ v.abs()
    delta = (q.numel() + 4) * 2.0 ** -24 * float((k.abs() @ q.abs()).max()) * scale
    return o, 2.0 ** -8 * o.abs() + 1.01 * (2.0 ** -16 + 2 * delta + 2.0 ** -20 + 2 * k.size(0) * 2.0 ** -24) * A + 1e-30


def compare(out, rows, what, f=attend_f32):
    """rows: (index into out [N, nh, hd], q, k, v)"""
    worst = 0.0
    for at, q, k, v in rows:
        o, tol = f(q, k, v, q.numel() ** -0.5)
        share = float(((out[at].double() - o).abs() / tol.clamp(min=1e-30)).max())
        assert share <= 1.0, (what, at, share)
        worst = max(worst, share)
    return worst


def packed_kv(c, every=1):
    nh, nkv, hd = c['heads']
    G, i = nh // nkv, 0
    for s, n in enumerate(c['lens']):
        for t in range(n):
            if t % every and t != n - 1:
                continue
            m = max(0, c['klen'][s] - (n - 1 - t))
            kv = c['cache'][s, :m].view(m, 2, nkv, hd)
            for h in sorted({0, (5 * t) % nh, nh - 1}):
                yield (i + t, h), c['qkv'][i + t, h * hd:(h + 1) * hd], kv[:, 0, h // G], kv[:, 1, h // G]
        i += n


def prefix_kv(c, every=1):
    nh, nkv, hd = c['heads']
    G = nh // nkv
    for i in range(0, c['B'] * c['T'], every):
        b, m = i // c['T'], c['klen'][i]
        x = c['P'] if c['plen'] is None else c['plen'][b]
        kv = torch.cat([c['prefix'][:x], c['cache'][b, :m]]).view(x + m, 2, nkv, hd)
        for h in sorted({0, (5 * i) % nh, nh - 1}):
            yield (i, h), c['qkv'][i, h * hd:(h + 1) * hd], kv[:, 0, h // G], kv[:, 1, h // G]


def run_packed(c, dev, split=True, **kw):
    from infernos_amd import ops
    nh, nkv, hd = c['heads']
    sizes = dict(ntokens=c['N'], nseqs=c['n'], nheads=nh, nkv=nkv, head_dim=hd, max_keys=c['max_keys'])
    out = torch.empty(c['N'], nh * hd, dtype=BF, device=dev)
    ops.attn_packed(c['qkv'], c['cache'], out, c['cu'], c['key_len'], max_pos=c['S'], ws=ops.attn_packed_ws(dev, **sizes) if split else None, **sizes, **kw)
    return out.view(c['N'], nh, hd)


def run_prefix(c, dev, **kw):
    from infernos_amd import ops
    nh, nkv, hd = c['heads']
    sizes = dict(nrows=c['B'], tokens_per_row=c['T'], prefix_keys=c['P'], nheads=nh, nkv=nkv, head_dim=hd, max_keys=c['max_keys'])
    out = torch.empty(c['B'] * c['T'], nh * hd, dtype=BF, device=dev)
    ops.attn_prefix(c['qkv'], c['prefix'], c['cache'], out, c['key_len'], max_pos=c['S'], prefix_len=c['prefix_len'],
                    ws=ops.attn_prefix_ws(dev, **sizes), **sizes, **kw)
    return out.view(c['B'] * c['T'], nh, hd)


# ---- the probabilities' bits -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize('heads,lens,past', [((4, 1, 64), [37, 1, 20], 0), ((12, 2, 128), [130, 41], 0), ((12, 2, 128), [33, 60], 1500),
                                             ((14, 2, 64), [1, 1, 2], 3000), ((12, 2, 128), [1] * 9, 200)])
def test_packed_probabilities_keep_16_bits(dev, heads, lens, past):
    """wide and narrow workgroups, keys whole and split; a caller may have the probabilities rounded to bf16 instead (2^-8 A more, with A
    of the tolerance above), which gives other bits"""
    c = packed_case(dev, heads, lens, [n + (past + 7 * s if past else 0) for s, n in enumerate(lens)], spare=3, seed=past + len(lens))
    rows = list(packed_kv(c, 9))
    for split in (True, False):
        out = run_packed(c, dev, split)
        print('packed', heads, lens, past, split, 'worst share of the tolerance %.2f' % compare(out, rows, 'packed'))
        rounded = run_packed(c, dev, split, probs_bf16=True)
        assert not torch.equal(out, rounded)
        compare(rounded, rows, 'rounded', rounded_tol)


@pytest.mark.parametrize('heads,B,T,P,own', [((4, 1, 64), 2, 1, 333, 40), ((12, 2, 128), 64, 1, 2048, 300), ((40, 8, 128), 64, 5, 1400, 400),
                                             ((14, 2, 64), 9, 3, 900, 300)])
def test_prefix_probabilities_keep_16_bits(dev, heads, B, T, P, own):
    """one launch and two, both key sets' forms"""
    c = prefix_case(dev, heads, B, T, P, [(b * 7919) % own for b in range(B)], seed=P)
    rows = list(prefix_kv(c, max(1, B * T // 40)))
    out = run_prefix(c, dev)
    print('prefix', heads, B, T, P, own, 'worst share of the tolerance %.2f' % compare(out, rows, 'prefix'))
    rounded = run_prefix(c, dev, probs_bf16=True)
    assert not torch.equal(out, rounded)
    compare(rounded, rows, 'rounded', rounded_tol)


def rounded_tol(q, k, v, scale):
    o, tol = attend_f32(q, k, v, scale)
    if k.size(0) == 0:
        return o, tol
    return o, tol + 2.0 ** -8 * (torch.softmax((k.double() @ q.double()) * scale, 0) @ v.double().abs())


# ---- scores at the ends of f32 ---------------------------------------------------------------------------------------------
def far_down(c):
    """scores of every key about -360 in front of the exponential (dimension 1), a first head_dim in which the first keys may be infinite"""
    nh, nkv, hd = c['heads']
    q = c['qkv'][:, :nh * hd].view(-1, nh, hd)
    q[..., 0], q[..., 1] = -1.0, 64.0
    q[..., 2:] *= 0.1


@pytest.mark.parametrize('heads,lens,past,split', [((4, 2, 128), [70], 130, False), ((4, 2, 128), [3], 3000, True), ((4, 1, 64), [1, 2], 700, False),
                                                   ((12, 2, 128), [200], 0, False)])
def test_packed_scores_of_minus_infinity_in_the_first_keys(dev, heads, lens, past, split):
    """keys whose score is -inf (an infinite K element against a negative q) fill more than the first tile of every wave: their weight is 0
    and the keys behind them keep theirs, however low their scores lie"""
    c = packed_case(dev, heads, lens, [n + past for n in lens], spare=2, seed=past)
    nh, nkv, hd = heads
    far_down(c)
    k = c['cache'][:, :, :nkv * hd].view(c['n'], c['S'], nkv, hd)
    k[..., 1] = -64.0
    k[:, :140 if past else 40, :, 0] = float('inf')
    skip = 140 if past else 40
    rows = [(at, q, kk[skip:], v[skip:]) for at, q, kk, v in packed_kv(c, 7) if kk.size(0) > skip]
    assert rows
    print('worst share %.2f' % compare(run_packed(c, dev, split), rows, 'minus infinity'))


def test_prefix_scores_of_minus_infinity_in_the_first_keys(dev):
    """the same in the shared keys, read in a launch with the own keys and in workgroups of their own"""
    for heads, B, T, P in (((4, 1, 64), 2, 1, 300), ((12, 2, 128), 24, 2, 2000)):
        c = prefix_case(dev, heads, B, T, P, [20 + b for b in range(B)], seed=P)
        nh, nkv, hd = heads
        far_down(c)
        for kv in (c['prefix'], c['cache']):
            kv.view(-1, kv.size(-1))[:, :nkv * hd].view(-1, nkv, hd)[..., 1] = -64.0
        c['prefix'][:140, :nkv * hd].view(140, nkv, hd)[..., 0] = float('inf')
        rows = [(at, q, k[140:], v[140:]) for at, q, k, v in prefix_kv(c, max(1, B * T // 8))]
        print('worst share %.2f' % compare(run_prefix(c, dev), rows, 'minus infinity'))


@pytest.mark.parametrize('past,split', [(0, False), (3000, True)])
def test_packed_scores_near_the_lowest_f32(dev, past, split):
    """scores of -1e34 and, for one key, half of that: its value is the result"""
    heads = nh, nkv, hd = (4, 1, 64)
    c = packed_case(dev, heads, [2], [2 + past + 50], seed=1)
    c['qkv'][:, :nh * hd] = 0.0
    c['qkv'][:, 0:nh * hd:hd] = 2.0 ** 58
    n = c['klen'][0]
    k = c['cache'][0, :n, :hd]
    k.zero_()
    k[:, 0] = -2.0 ** 58
    at = n // 2
    k[at, 0] = -2.0 ** 57
    out = run_packed(c, dev, split)
    assert torch.equal(out, c['cache'][0, at, hd:].expand_as(out))
    x = prefix_case(dev, heads, 2, 1, n, [40, 50], seed=2)
    x['qkv'][:, :nh * hd] = c['qkv'][:2, :nh * hd]
    x['prefix'] = c['cache'][0, :n].contiguous()
    x['cache'][:, :, :hd] = 0.0
    x['cache'][:, :, 0] = -2.0 ** 58
    out = run_prefix(x, dev)
    assert torch.equal(out, c['cache'][0, at, hd:].expand_as(out))


# ---- every form of the shared-prefix launch --------------------------------------------------------------------------------
JOINT, TWO, BOTH, NARROW_PREFIX, NARROW_OWN = 0, 1, 2, 4, 8


@pytest.mark.parametrize('heads,B,T,P,own,form', [((14, 2, 64), 64, 3, 4000, 620, BOTH + NARROW_OWN), ((14, 2, 64), 128, 6, 1500, 300, BOTH),
                                                  ((8, 8, 64), 96, 6, 2500, 90, BOTH + NARROW_OWN), ((16, 2, 64), 70, 5, 3001, 1100, BOTH),
                                                  ((40, 8, 128), 40, 7, 1500, 2000, BOTH), ((12, 2, 128), 160, 1, 6000, 700, BOTH + NARROW_OWN),
                                                  ((14, 2, 64), 20, 6, 900, 300, TWO + NARROW_PREFIX), ((14, 2, 64), 9, 1, 2000, 300, TWO + NARROW_PREFIX + NARROW_OWN),
                                                  ((12, 2, 128), 3, 7, 1500, 700, TWO + NARROW_PREFIX), ((40, 8, 128), 9, 7, 900, 200, TWO),
                                                  ((12, 2, 128), 96, 1, 2048, 300, TWO + NARROW_OWN),
                                                  ((4, 1, 64), 5, 2, 500, 90, JOINT + NARROW_OWN)])
def test_prefix_forms(dev, heads, B, T, P, own, form):
    """the form that the sizes ask for, its rows of every kind: without an own key, with a part of the prefix or none of it"""
    from infernos_amd import _lib
    plen = [0 if b % 11 == 3 else P if b % 4 else 1 + (P * 7 * b) % P for b in range(B)]
    lens = [-1 if b % 13 == 5 else (b * 7919) % (own + 1) for b in range(B)]
    lens[0] = own
    c = prefix_case(dev, heads, B, T, P, lens, plen=plen, seed=own)
    assert _lib.lib().ifh_attn_prefix_form(B, T, P, heads[0], heads[1], c['max_keys']) == form
    w = compare(run_prefix(c, dev), list(prefix_kv(c, max(1, B * T // 60))), 'prefix')
    compare(run_prefix(c, dev, probs_bf16=True), list(prefix_kv(c, max(1, B * T // 30))), 'rounded', rounded_tol)
    print('attn_prefix ok', heads, B, T, P, own, 'form', form, 'worst share %.2f' % w)


# ---- draft verification: borders -------------------------------------------------------------------------------------------
def run_verify(dev, logits, drafts, u, V, temperature, q=None, ld=None, q_ld=None, lens=None):
    from infernos_amd import ops
    B, T1 = u.shape
    tok, cnt = torch.full((B, T1), -7, dtype=torch.int32, device=dev), torch.full((B,), -7, dtype=torch.int32, device=dev)
    ws = ops.verify_drafts_ws(B, T1 - 1, dev)
    ws.fill_(255)
    ops.verify_drafts(logits, drafts, u, tok, cnt, ws, vocab=V, ld=V if ld is None else ld, nrows=B, ndraft=T1 - 1, temperature=temperature,
                      draft_probs=q, q_ld=q_ld, lens=lens)
    return tok, cnt


@pytest.mark.parametrize('temp', [0.7, 1.3, 0.1])
def test_the_temperature_is_the_callers_double(dev, temp):
    """uniform numbers that lie between a border of softmax(logits / temp) and the same border with the temperature rounded to f32 (up to
    5e-8 away), 2e-9 or more from the first: the token is the one of the caller's temperature.  (The masses are good to 1e-10.)"""
    V, B = 4096, 400
    g = torch.Generator(device=dev).manual_seed(7)
    logits = torch.randn(B, V, generator=g, device=dev) * min(2.0, 2.0 * temp)
    # (on the CPU: the device's softmax of f64 tensors is off by 1e-8)
    c = [torch.softmax(logits.cpu().double() / t, 1).cumsum(1).to(dev) for t in (temp, float(torch.tensor(temp, dtype=torch.float32)))]
    mid = (c[0] + c[1]) / 2
    u = mid.float()
    between = (u.double() - c[0]).sign() * (u.double() - c[1]).sign() < 0
    ok = between & ((u.double() - c[0]).abs() > 2e-9) & (u < 1)
    rows = ok.any(1)
    at = ok.float().argmax(1)
    u = u.gather(1, at[:, None])[rows].contiguous()
    logits, c = logits[rows].contiguous(), c[0][rows]
    want = torch.searchsorted(c, u.double(), right=True)[:, 0]
    assert want.numel() >= 50
    tok, cnt = run_verify(dev, logits, torch.zeros(1, 1, dtype=torch.int32, device=dev), u, V, temp)
    assert torch.equal(tok[:, 0].long(), want), int((tok[:, 0].long() != want).sum())


def test_masses_keep_the_bits_of_f64(dev):
    """two tokens of logits 0 and d: the first is drawn while u (1 + e^d) < 1.  Of four million d those whose f32 number nearest to the
    border lies within 3e-12 of it, but 2e-14 or more away (80-bit exponentials; f64 masses, their sum and the product are good to
    1e-15): an exponential that is 1e-11 off takes the other token of many"""
    import numpy as np
    d = -np.arange(1 << 22, dtype=np.float64) * 2.0 ** -22 - 2.0 ** -23                     # exact in f32
    e = np.exp(d.astype(np.longdouble))
    u = (1 / (1 + e)).astype(np.float32)
    gap = (u.astype(np.longdouble) * (1 + e) - 1).astype(np.float64)
    at = np.nonzero((np.abs(gap) < 3e-12) & (np.abs(gap) > 2e-14))[0]
    assert at.size > 100 and np.finfo(np.longdouble).eps < 1e-18 and (d.astype(np.float32) == d).all()
    logits = torch.tensor(np.stack([np.zeros(at.size), d[at]], 1), dtype=torch.float32, device=dev)
    want = torch.tensor(gap[at] > 0, device=dev).long()
    tok, _ = run_verify(dev, logits, torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.tensor(u[at], device=dev)[:, None].contiguous(), 2, 1.0)
    wrong = int((tok[:, 0].long() != want).sum())
    assert wrong == 0, (wrong, at.size)


def test_a_chunk_without_mass_is_not_drawn_from(dev):
    """one token in each of the chunks 0, 1, 2 and 4 of 2048, of masses 2^-53, 2^-53, 1 and 1 (at this temperature a logit of -53 is exactly
    that), nothing in chunk 3.  ((0 + 1) + (2^-53 + 2^-53)) is a bit more than ((1 + 2^-53) + 2^-53), so a sum up to chunk 3 may lie
    above the number 1 that the draw looks for and the sum up to chunk 2 not: the token comes from a chunk that has one all the same"""
    V = 5 * 2048
    logits = torch.full((1, V), -float('inf'), device=dev)
    at = [5, 2048 + 700, 4096 + 1, 8192 + 2047]
    logits[0, at] = torch.tensor([-53.0, -53.0, 0.0, 0.0], device=dev)
    tok, cnt = run_verify(dev, logits, torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.tensor([[0.5]], device=dev), V, 1.4426950408889634)
    assert int(tok[0, 0]) in at[2:] and int(cnt[0]) == 1, tok


# ---- draft verification: a server's batches --------------------------------------------------------------------------------
# A chunk is 2048 logits.  A wave takes a chunk of the statistics where there are more than 32 chunks a CU, and of the remaining mass where
# more than 12, else four waves do; on 256 CUs: (64, 4, 151936) 94 and 19, (600, 2, 14337) 56 and 19, (500, 2, 8193) 29 and 10, (1100, 1,
# 8000) 34 and 17, (2, 3, 151936) 2 and 1.
@pytest.mark.parametrize('B,T,V', [(64, 4, 151936), (600, 2, 14337), (500, 2, 8193), (1100, 1, 8000), (2, 3, 151936)])
@pytest.mark.parametrize('pad,q_pad,temp', [(0, 0, 0.7), (0, None, 1.0), (3, 3, 1.3), (3, None, 0.7), (4, 3, 0.7), (3, 4, 1.0), (0, None, 0.0), (3, 0, 0.0)])
def test_verify_batches(dev, B, T, V, pad, q_pad, temp):
    """both kernel forms, several chunks a row and the last one in part, rows of logits and of the draft's distribution aligned and not
    (q_pad None: looked-up drafts), a draft count for each row; some rows in 64 bits on the CPU"""
    g = torch.Generator(device=dev).manual_seed(B + V + pad)
    ld = -(-V // 4) * 4 + pad
    logits = torch.full((B * (T + 1), ld), 50.0, device=dev)                     # (columns behind the vocabulary are not used)
    logits[:, :V] = torch.randn(B * (T + 1), V, generator=g, device=dev) * 2
    at = torch.randint(0, V, (B * (T + 1), 6), generator=g, device=dev)
    logits.scatter_(1, at, 9.0 + torch.rand(at.shape, generator=g, device=dev))
    logits[:, V - 1] = 8.0
    t = temp or 1.0
    q = q_ld = None
    if q_pad is not None:
        q_ld = -(-V // 4) * 4 + q_pad
        q = torch.full((B * T, q_ld), 0.5, device=dev)
        near = logits.view(B, T + 1, ld)[:, :T, :V].reshape(B * T, V) + 0.3 * torch.randn(B * T, V, generator=g, device=dev)
        q[:, :V] = torch.softmax(near / t, 1)
        drafts = torch.multinomial(q[:, :V], 1, generator=g).view(B, T)
        del near
    else:
        pick = torch.randint(0, 6, (B, T, 1), generator=g, device=dev)
        drafts = at.view(B, T + 1, 6)[:, :T].gather(2, pick)[:, :, 0]
    drafts = drafts.to(torch.int32).contiguous()
    if temp == 0:
        logits.view(B, T + 1, ld)[:, :, 77] = 11.0                              # ties: the lowest id
        logits.view(B, T + 1, ld)[::2, :, V - 1] = 11.0
        drafts[::3] = 77
    u = torch.rand(B, T + 1, generator=g, device=dev)
    lens = [T - (r % 7 == 3) for r in range(B)]
    tok, cnt = run_verify(dev, logits, drafts, u, V, temp, q, ld, q_ld, i32(lens, dev))
    tok, cnt = tok.cpu(), cnt.cpu()
    seen = set()
    for r in sorted({0, B - 1, *range(1, B, max(1, B // 9))}):
        l = logits[r * (T + 1):(r + 1) * (T + 1), :V].cpu().double()
        d = drafts[r].cpu()
        if temp == 0:
            p = torch.nn.functional.one_hot((l == l.max(1, keepdim=True).values).to(torch.int8).argmax(1), V).double()
        else:
            p = torch.softmax(l / temp, 1)
        qr = q[r * T:(r + 1) * T, :V].cpu().double() if q is not None else torch.nn.functional.one_hot(d.long(), V).double()
        kept, mass, margin = verify64(p, qr, d, u[r].cpu(), lens[r])
        assert margin > 1e-10
        check_verified(tok, cnt, r, kept, mass, d, float(u[r, T]))
        seen.add(kept)
    print('verify ok', B, T, V, pad, q_pad, temp, 'kept', sorted(seen))
