"""The operators that serve the language model's prompts and decode steps beyond one padded batch, as cases to be measured:

  packed   causal grouped-query attention of prompts laid end to end, each against its own cache row
  prefix   grouped-query attention of a decode step whose rows share one long prefix (a system prompt kept once)
  rope     rotary embedding and KV append of tokens laid end to end
  verify   verification of drafted tokens against the target's distribution, from given uniform numbers

With `own` false, run() computes them in elementary torch operations in 32 bits (64 for the draws); with `own` true it makes the
calls of infernos_amd.ops that a program makes.  exact() gives the same results in 64 bits, from the definitions.
"""
import math
import random

import torch

own = False

BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
DEV = 'cuda'
CAND = 32                       # candidates a row of the top-k sampler keeps


# ---- cases --------------------------------------------------------------------------------------------------------------
def _packed(name, nseq, new, past, heads, seed):
    return dict(name=name, op='packed', nseq=nseq, new_lo=new[0], new_hi=new[1], past_lo=past[0], past_hi=past[1], nh=heads[0],
                nkv=heads[1], hd=heads[2], lens=seed)


def _prefix(name, nrows, tokens, prefix, past, heads, seed, part=0):
    return dict(name=name, op='prefix', nrows=nrows, tokens=tokens, prefix=prefix, past_lo=past[0], past_hi=past[1], nh=heads[0],
                nkv=heads[1], hd=heads[2], part=part, lens=seed)


def _rope(name, nseq, new, past, heads, seed):
    return dict(_packed(name, nseq, new, past, heads, seed), op='rope')


def _verify(name, form, nrows, ndraft, vocab, probs, temperature, seed):
    return dict(name=name, op='verify', form=form, nrows=nrows, ndraft=ndraft, vocab=vocab, probs=probs, temperature=temperature, lens=seed)


SMALL, GROUP6, WIDE = (4, 1, 64), (12, 2, 128), (40, 8, 128)         # query heads, kv heads, head_dim


def listed():
    return [
        # three short utterances reach an idle server together: latency
        _packed('packed 3 short prompts', 3, (1, 40), (0, 0), SMALL, 1),
        # a batch of sessions' first prompts, every length its own
        _packed('packed 64 prompts', 64, (40, 320), (0, 0), GROUP6, 2),
        # the next turn of eight calls: new text behind what their cache rows hold
        _packed('packed 8 turns on a cache', 8, (33, 257), (1000, 4000), GROUP6, 3),
        # one long document in a single pass
        _packed('packed one long prompt', 1, (8191, 8191), (0, 0), WIDE, 4),
        # two calls behind a short system prompt: latency
        _prefix('prefix 2 rows', 2, 1, 333, (1, 40), SMALL, 5),
        # a decode step of 64 calls that share a system prompt
        _prefix('prefix 64 rows', 64, 1, 2048, (16, 512), GROUP6, 6),
        # the same step with four drafted tokens a row, behind a long shared document, some rows using a part of it
        _prefix('prefix 64 rows 5 tokens', 64, 5, 8001, (100, 1500), WIDE, 7, part=1),
        # the tokens of one decode step of two rows with a draft each: latency
        _rope('rope 2 drafts', 2, (2, 5), (10, 300), SMALL, 8),
        # the append of a batch of prompts
        _rope('rope 64 prompts', 64, (40, 320), (0, 500), GROUP6, 9),
        # the draft step of 64 calls under top-k / top-p sampling
        _verify('verify top-k 64 rows', 'topk', 64, 4, 151936, 1, 0.7, 10),
        # one call, drafts from a lookup (no distribution of their own): latency
        _verify('verify 1 row lookup', 'full', 1, 3, 151936, 0, 1.0, 11),
        # 64 calls, drafts of a small model with its whole distribution
        _verify('verify 64 rows', 'full', 64, 4, 151936, 1, 0.8, 12),
    ]


HEADS = (SMALL, (4, 2, 128), GROUP6, (14, 2, 64), WIDE, (8, 8, 64), (16, 1, 128))


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _cost(case):
    w = work(case)
    return max(w['bytes'], w['flops'] / 50)


def _plain_elems(case):
    """elements of the plain form's score matrix"""
    if case['op'] == 'packed':
        return case['nseq'] * case['new_hi'] * (case['new_hi'] + case['past_hi']) * case['nh']
    if case['op'] == 'prefix':
        return case['nrows'] * case['tokens'] * (case['prefix'] + case['past_hi'] + case['tokens']) * case['nh']
    return 0


def draw(rng):
    big = listed()
    while True:
        op = rng.choice(('packed', 'packed', 'prefix', 'prefix', 'rope', 'verify'))
        heads, seed = rng.choice(HEADS), rng.randrange(1 << 20)
        if op in ('packed', 'rope'):
            n, hi = _log(rng, 1, 96), _log(rng, 1, 8191)
            past = _log(rng, 1, 8191) if rng.random() < 0.5 else 0
            c = (_packed if op == 'packed' else _rope)('', n, (max(1, hi // 8), hi), (past // 4, past), heads, seed)
        elif op == 'prefix':
            hi = _log(rng, 1, 2047)
            c = _prefix('', _log(rng, 1, 96), rng.randint(1, 6), _log(rng, 1, 16001), (hi // 6, hi), heads, seed, part=rng.randint(0, 1))
        else:
            form = rng.choice(('full', 'full', 'topk'))
            c = _verify('', form, _log(rng, 1, 96), rng.randint(1, 6), rng.choice((777, 1000, 32003, 151936, 152064)),
                        rng.randint(0, 1), rng.choice((0.5, 0.7, 1.0, 1.3)), seed)
        del c['name']
        if _cost(c) <= max(_cost(b) for b in big if b['op'] == op) and _plain_elems(c) <= max(_plain_elems(b) for b in big):
            return c


def _lens(case):
    """new tokens and tokens already in the cache, a sequence each: part of the case, not of the seed"""
    r = random.Random(case['lens'])
    if case['op'] == 'prefix':
        return [case['tokens']] * case['nrows'], [r.randint(case['past_lo'], case['past_hi']) for _ in range(case['nrows'])]
    return ([r.randint(case['new_lo'], case['new_hi']) for _ in range(case['nseq'])],
            [r.randint(case['past_lo'], case['past_hi']) for _ in range(case['nseq'])])


def _prefix_lens(case):
    r = random.Random(case['lens'] + 1)
    return [case['prefix'] if not case['part'] or r.random() < 0.75 else r.randint(0, case['prefix']) for _ in range(case['nrows'])]


def work(case):
    op = case['op']
    if op == 'verify':
        rows, T = case['nrows'], case['ndraft']
        if case['form'] == 'topk':
            n = rows * (T + 1) * CAND * 8 + (rows * T * CAND * 8 if case['probs'] else 0)
            return dict(bytes=n + rows * (3 * T + 3) * 4, flops=rows * (2 * T + 1) * CAND * 4)
        n = rows * (T + 1) * case['vocab']
        q = rows * case['vocab'] if case['probs'] else 0             # the draft's distribution at the one position that is drawn
        return dict(bytes=4 * (n + q) + rows * (3 * T + 3) * 4, flops=4 * n + 6 * q)
    new, past = _lens(case)
    nh, nkv, hd = case['nh'], case['nkv'], case['hd']
    N = sum(new)
    if op == 'rope':
        pos = max(n + p for n, p in zip(new, past))
        return dict(bytes=2 * 2 * N * (nh + 2 * nkv) * hd + 4 * min(N, pos) * hd, flops=3 * N * (nh + nkv) * hd)
    io = 2 * 2 * N * nh * hd
    if op == 'packed':
        keys = sum(n + p for n, p in zip(new, past))
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    else:
        pl = _prefix_lens(case)
        keys = max(pl) + sum(n + p for n, p in zip(new, past))
        pairs = sum(n * (p + x) + n * (n + 1) // 2 for n, p, x in zip(new, past, pl))
    return dict(bytes=io + keys * 2 * nkv * hd * 2, flops=4 * pairs * nh * hd)


# ---- inputs -------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def _logits(g, rows, vocab):
    """a language model's logits: a broad bulk and a few tokens that stand out of it"""
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 2.0
    at = torch.randint(0, vocab, (rows, 24), generator=g, device=DEV)
    return x.scatter_add_(1, at, torch.rand(rows, 24, generator=g, device=DEV) * 12.0 + 4.0)


def _draw_rows(p, g):
    c = p.double().cumsum(1)
    u = torch.rand(p.size(0), 1, generator=g, device=DEV, dtype=F64) * c[:, -1:]
    return torch.searchsorted(c, u, right=True).clamp_(max=p.size(1) - 1)


def _nucleus(logits, temperature, k=20, top_p=0.8):
    """the top-k sampler's candidates of each row, best first, and their final probabilities (0: dropped)"""
    v, i = (logits / temperature).topk(min(CAND, logits.size(1)), dim=1)
    p = torch.softmax(v.double().masked_fill(torch.arange(v.size(1), device=DEV) >= k, -math.inf), 1)
    below = p.flip(1).cumsum(1).flip(1)                              # the mass of a candidate and everything below it
    keep = below > 1 - top_p
    keep[:, 0] = True
    p = p * keep
    return i.to(I32).contiguous(), (p / p.sum(1, keepdim=True)).float().contiguous()


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=case, ws=None)
    rnd = lambda *n: torch.randn(*n, generator=g, device=DEV)
    if case['op'] == 'verify':
        rows, T, V = case['nrows'], case['ndraft'], case['vocab']
        t = _logits(g, rows * (T + 1), V)
        d = (t.view(rows, T + 1, V)[:, :T] + rnd(rows, T, V) * 0.7).reshape(rows * T, V)          # a smaller model's view of the same text
        if case['form'] == 'topk':
            s['cand'], s['prob'] = _nucleus(t, case['temperature'])
            dc, dp = _nucleus(d, case['temperature'])
            at = _draw_rows(dp, g)
            s['drafts'] = dc.gather(1, at).view(rows, T).contiguous()
            s['dcand'], s['dprob'] = (dc, dp) if case['probs'] else (None, None)
        else:
            s['logits'] = t
            q = torch.softmax(d / case['temperature'], 1)
            s['drafts'] = _draw_rows(q, g).to(I32).view(rows, T).contiguous()
            s['q'] = q.contiguous() if case['probs'] else None
        s['uniform'] = torch.rand(rows, T + 1, generator=g, device=DEV)
        s['tokens'] = torch.empty(rows, T + 1, dtype=I32, device=DEV)
        s['count'] = torch.empty(rows, dtype=I32, device=DEV)
        return s
    new, past = _lens(case)
    nh, nkv, hd = case['nh'], case['nkv'], case['hd']
    N, n = sum(new), len(new)
    S = -(-max(a + b for a, b in zip(new, past)) // 16) * 16
    cu = [0]
    for a in new:
        cu.append(cu[-1] + a)
    s.update(N=N, n=n, S=S, max_new=max(new), max_keys=max(a + b for a, b in zip(new, past)), cu=_i32(cu))
    s['qkv'] = rnd(N, (nh + 2 * nkv) * hd)
    s['qkv'][:, :nh * hd] *= 2.0                                     # scores that tell keys apart
    s['qkv'] = s['qkv'].to(BF16)
    s['cache'] = rnd(n, S, 2 * nkv * hd).to(BF16)
    if case['op'] == 'rope':
        P = max(a + b for a, b in zip(new, past))
        ang = torch.arange(P, device=DEV, dtype=F64)[:, None] * (1.0e6 ** (-torch.arange(0, hd, 2, device=DEV, dtype=F64) / hd))[None]
        s['cs'] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
        s['pos0'] = _i32(past)
        s['q'] = torch.empty(N, nh * hd, dtype=BF16, device=DEV)
        return s
    s['out'] = torch.empty(N, nh * hd, dtype=BF16, device=DEV)
    if case['op'] == 'packed':
        s['key_len'] = _i32([a + b for a, b in zip(new, past)])
    else:
        s['prefix'] = rnd(case['prefix'], 2 * nkv * hd).to(BF16)
        s['prefix_len'] = _i32(_prefix_lens(case)) if case['part'] else None
        s['key_len'] = _i32([p + t + 1 for a, p in zip(new, past) for t in range(a)])
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------------
def _token_places(s):
    """for every packed token: its sequence and its place within it"""
    i = torch.arange(s['N'], device=DEV)
    seq = torch.searchsorted(s['cu'][1:].contiguous(), i.to(I32), right=True)
    return seq, i - s['cu'].long()[seq]


def _softmax_times(scores, visible, v):
    """softmax over the visible keys, times v; a row that sees nothing gives zeros"""
    scores = scores.masked_fill_(~visible, -math.inf)
    m = scores.amax(-1, keepdim=True)
    w = scores.sub_(torch.where(m > -math.inf, m, 0)).exp_()
    l = w.sum(-1, keepdim=True)
    return torch.matmul(w, v) / torch.where(l > 0, l, 1)


def _plain_packed(s):
    c = s['case']
    nh, nkv, hd, n, T, K = c['nh'], c['nkv'], c['hd'], s['n'], s['max_new'], s['max_keys']
    G = nh // nkv
    seq, t = _token_places(s)
    q = torch.zeros(n, T, nkv, G, hd, device=DEV)
    q[seq, t] = s['qkv'][:, :nh * hd].float().view(-1, nkv, G, hd)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, nkv, G * T, hd)
    kv = s['cache'][:, :K].float().view(n, K, 2, nkv, hd)
    k = kv[:, :, 0].permute(0, 2, 3, 1).contiguous()
    v = kv[:, :, 1].permute(0, 2, 1, 3).contiguous()
    lens = s['cu'][1:] - s['cu'][:-1]
    see = (s['key_len'] - lens)[:, None] + torch.arange(1, T + 1, device=DEV)                     # keys each query sees
    visible = torch.arange(K, device=DEV) < see[:, :, None]
    visible = visible[:, None, None].expand(n, 1, G, T, K).reshape(n, 1, G * T, K)
    o = _softmax_times(torch.matmul(q, k).mul_(hd ** -0.5), visible, v)
    o = o.view(n, nkv, G, T, hd).permute(0, 3, 1, 2, 4)[seq, t]
    s['out'].copy_(o.reshape(s['N'], nh * hd))
    return s['out']


def _plain_prefix(s):
    c = s['case']
    nh, nkv, hd, B, T, P, K = c['nh'], c['nkv'], c['hd'], c['nrows'], c['tokens'], c['prefix'], s['max_keys']
    G = nh // nkv
    q = s['qkv'][:, :nh * hd].float().view(B, T, nkv, G, hd)
    pk = s['prefix'].float().view(P, 2, nkv, hd)
    ck = s['cache'][:, :K].float().view(B, K, 2, nkv, hd)
    qp = q.permute(2, 0, 1, 3, 4).reshape(nkv, B * T * G, hd).contiguous()
    sp = torch.matmul(qp, pk[:, 0].permute(1, 2, 0).contiguous()).view(nkv, B, T, G, P).permute(1, 0, 2, 3, 4)
    qo = q.permute(0, 2, 1, 3, 4).reshape(B, nkv, T * G, hd).contiguous()
    so = torch.matmul(qo, ck[:, :, 0].permute(0, 2, 3, 1).contiguous()).view(B, nkv, T, G, K)
    scores = torch.cat([sp, so], -1).mul_(hd ** -0.5)
    plen = s['prefix_len'] if s['prefix_len'] is not None else torch.full((B,), P, device=DEV)
    vis_p = (torch.arange(P, device=DEV) < plen[:, None])[:, None, None, None, :].expand(B, nkv, T, G, P)
    vis_o = (torch.arange(K, device=DEV) < s['key_len'].view(B, T)[:, :, None])[:, None, :, None, :].expand(B, nkv, T, G, K)
    scores = scores.masked_fill_(~torch.cat([vis_p, vis_o], -1), -math.inf)
    m = scores.amax(-1, keepdim=True)
    w = scores.sub_(torch.where(m > -math.inf, m, 0)).exp_()
    l = w.sum(-1, keepdim=True)
    wp = w[..., :P].permute(1, 0, 2, 3, 4).reshape(nkv, B * T * G, P)
    o = torch.matmul(wp, pk[:, 1].permute(1, 0, 2).contiguous()).view(nkv, B, T, G, hd).permute(1, 0, 2, 3, 4)
    o = o + torch.matmul(w[..., P:].reshape(B, nkv, T * G, K), ck[:, :, 1].permute(0, 2, 1, 3).contiguous()).view(B, nkv, T, G, hd)
    o = o / torch.where(l > 0, l, 1)
    s['out'].copy_(o.permute(0, 2, 1, 3, 4).reshape(B * T, nh * hd))
    return s['out']


def _plain_rope(s):
    c = s['case']
    nh, nkv, hd = c['nh'], c['nkv'], c['hd']
    seq, t = _token_places(s)
    pos = s['pos0'].long()[seq] + t
    x = s['qkv'].float().view(s['N'], nh + 2 * nkv, hd)
    cos, sin = s['cs'][pos][:, None, :, 0], s['cs'][pos][:, None, :, 1]
    a, b = x[:, :nh + nkv, :hd // 2], x[:, :nh + nkv, hd // 2:]
    r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(BF16)
    s['q'].copy_(r[:, :nh].reshape(s['N'], -1))
    s['cache'][seq, pos] = torch.cat([r[:, nh:].reshape(s['N'], -1), s['qkv'][:, (nh + nkv) * hd:]], 1)
    return s['q'], s['cache']


def _finish(drafts, accepted, token):
    """accepted drafts, the drawn token behind them, -1 to the end"""
    rows, T = drafts.shape
    i = torch.arange(T + 1, device=drafts.device)
    padded = torch.cat([drafts.long(), drafts.new_zeros(rows, 1).long()], 1)
    out = torch.where(i < accepted[:, None], padded, torch.where(i == accepted[:, None], token[:, None], -1))
    return out.to(I32), (accepted + 1).to(I32)


def _plain_verify(s):
    c = s['case']
    rows, T = c['nrows'], c['ndraft']
    drafts, u = s['drafts'], s['uniform'].double()
    if c['form'] == 'topk':
        p = s['prob'].double().view(rows, T + 1, -1)
        cand = s['cand'].view(rows, T + 1, -1)
        px = (p[:, :T] * (cand[:, :T] == drafts[:, :, None])).sum(-1)
        if s['dprob'] is not None:
            dp, dc = s['dprob'].double().view(rows, T, -1), s['dcand'].view(rows, T, -1)
            qx = (dp * (dc == drafts[:, :, None])).sum(-1)
            q = (dp[:, :, None, :] * (dc[:, :, None, :] == cand[:, :T, :, None])).sum(-1)
        else:
            qx, q = torch.ones_like(px), (cand[:, :T] == drafts[:, :, None]).double()
    else:
        V = c['vocab']
        p = torch.softmax(s['logits'].view(rows, T + 1, V).double() / c['temperature'], -1)
        cand = None
        x = drafts.long()[:, :, None]
        px = p[:, :T].gather(2, x)[:, :, 0]
        if s['q'] is not None:
            q = s['q'].view(rows, T, V)
            qx = q.gather(2, x)[:, :, 0].double()
        else:
            qx = torch.ones_like(px)
    ok = (u[:, :T] * qx < px).to(torch.int64)
    a = ok.cumprod(1).sum(1)                                         # drafts accepted before the first refusal
    r = torch.arange(rows, device=DEV)
    w = p[r, a]
    at = a.clamp(max=T - 1)
    if c['form'] == 'topk' or s['q'] is not None:
        minus = q[r, at].double()
    else:
        minus = torch.zeros_like(w).scatter_(1, drafts.long()[r, at][:, None], 1.0)
    rest = (w - minus).clamp(min=0)
    w = torch.where(((a < T) & (rest.sum(1) > 0))[:, None], rest, w)
    cum = w.cumsum(1)
    j = (cum > u[:, T:] * cum[:, -1:]).to(torch.int8).argmax(1)      # the first whose cumulated mass passes the uniform number
    token = j if cand is None else cand[r, a].long().gather(1, j[:, None])[:, 0]
    tokens, count = _finish(drafts, a, token)
    s['tokens'].copy_(tokens)
    s['count'].copy_(count)
    return s['tokens'], s['count']


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _own(s):
    from infernos_amd import ops
    c = s['case']
    if c['op'] == 'verify':
        if c['form'] == 'topk':
            ops.verify_drafts_topk(s['cand'], s['prob'], s['drafts'], s['uniform'], s['tokens'], s['count'], nrows=c['nrows'],
                                   ndraft=c['ndraft'], draft_cand=s['dcand'], draft_probs=s['dprob'])
        else:
            if s['ws'] is None:
                s['ws'] = ops.verify_drafts_ws(c['nrows'], c['ndraft'], DEV)
            ops.verify_drafts(s['logits'], s['drafts'], s['uniform'], s['tokens'], s['count'], s['ws'], vocab=c['vocab'], ld=c['vocab'],
                              nrows=c['nrows'], ndraft=c['ndraft'], temperature=c['temperature'], draft_probs=s['q'])
        return s['tokens'], s['count']
    heads = dict(nheads=c['nh'], nkv=c['nkv'], head_dim=c['hd'], max_pos=s['S'])
    if c['op'] == 'rope':
        ops.rope_append_packed(s['qkv'], s['cs'], s['cache'], s['cu'], s['pos0'], ntokens=s['N'], nseqs=s['n'], q_out=s['q'], **heads)
        return s['q'], s['cache']
    if c['op'] == 'packed':
        if s['ws'] is None:
            s['ws'] = ops.attn_packed_ws(DEV, ntokens=s['N'], nseqs=s['n'], nheads=c['nh'], nkv=c['nkv'], head_dim=c['hd'], max_keys=s['max_keys'])
        return ops.attn_packed(s['qkv'], s['cache'], s['out'], s['cu'], s['key_len'], ntokens=s['N'], nseqs=s['n'],
                               max_keys=s['max_keys'], ws=s['ws'], **heads)
    if s['ws'] is None:
        s['ws'] = ops.attn_prefix_ws(DEV, nrows=c['nrows'], tokens_per_row=c['tokens'], prefix_keys=c['prefix'], nheads=c['nh'],
                                     nkv=c['nkv'], head_dim=c['hd'], max_keys=s['max_keys'])
    return ops.attn_prefix(s['qkv'], s['prefix'], s['cache'], s['out'], s['key_len'], nrows=c['nrows'], tokens_per_row=c['tokens'],
                           prefix_keys=c['prefix'], max_keys=s['max_keys'], prefix_len=s['prefix_len'], ws=s['ws'], **heads)


def run(s):
    if own:
        return _own(s)
    return {'packed': _plain_packed, 'prefix': _plain_prefix, 'rope': _plain_rope, 'verify': _plain_verify}[s['case']['op']](s)


# ---- 64 bits, from the definitions, a sequence / a row at a time ------------------------------------------------------------
def _attend64(q, k, v, visible):
    """q [n, d], k and v [m, d], visible [n, m]"""
    z = (q @ k.t()) / math.sqrt(q.size(1))
    z = torch.where(visible, z, torch.full_like(z, -math.inf))
    p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)               # a row without a visible key: nothing
    return p @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'verify':
        return _exact_verify(case, s)
    new, past = _lens(case)
    nh, nkv, hd = case['nh'], case['nkv'], case['hd']
    G, x = nh // nkv, s['qkv'].double().view(s['N'], nh + 2 * nkv, hd)
    if case['op'] == 'rope':
        cache, q, i = s['cache'].double(), torch.empty(s['N'], nh * hd, dtype=F64, device=DEV), 0
        for b, (n, p) in enumerate(zip(new, past)):
            z = torch.view_as_complex(s['cs'][p:p + n].double().contiguous())[:, None]           # cos + i sin of each position and pair
            y = torch.complex(x[i:i + n, :nh + nkv, :hd // 2], x[i:i + n, :nh + nkv, hd // 2:]) * z
            y = torch.cat([y.real, y.imag], -1)
            q[i:i + n] = y[:, :nh].reshape(n, -1)
            cache[b, p:p + n, :nkv * hd] = y[:, nh:].reshape(n, -1)
            cache[b, p:p + n, nkv * hd:] = x[i:i + n, nh + nkv:].reshape(n, -1)
            i += n
        return q, cache
    out, i = torch.empty(s['N'], nh, hd, dtype=F64, device=DEV), 0
    pl = _prefix_lens(case) if case['op'] == 'prefix' else None
    for b, (n, p) in enumerate(zip(new, past)):
        m, at = n + p, torch.arange(n, device=DEV)
        kv = s['cache'][b, :m].double().view(m, 2, nkv, hd)
        seen = torch.arange(m, device=DEV)[None] <= p + at[:, None]
        if pl is not None:
            kv = torch.cat([s['prefix'][:pl[b]].double().view(pl[b], 2, nkv, hd), kv])
            seen = torch.cat([torch.ones(n, pl[b], dtype=torch.bool, device=DEV), seen], 1)
        for h in range(nh):
            out[i:i + n, h] = _attend64(x[i:i + n, h], kv[:, 0, h // G], kv[:, 1, h // G], seen)
        i += n
    return out.view(s['N'], nh * hd)


def _exact_verify(case, s):
    """drafts one by one: kept while the uniform number is below p / q; at the first refusal a draw from what p has over q, behind the
    last draft a draw from p"""
    rows, T = case['nrows'], case['ndraft']
    tokens, count = torch.full((rows, T + 1), -1, dtype=I32), torch.zeros(rows, dtype=I32)
    for r in range(rows):
        for i in range(T + 1):
            if case['form'] == 'topk':
                ids = s['cand'][r * (T + 1) + i].tolist()
                p = dict(zip(ids, s['prob'][r * (T + 1) + i].double().tolist()))
                if i < T:
                    x = int(s['drafts'][r, i])
                    q = dict(zip(s['dcand'][r * T + i].tolist(), s['dprob'][r * T + i].double().tolist())) if case['probs'] else {x: 1.0}
                    if float(s['uniform'][r, i]) * q.get(x, 0.0) < p.get(x, 0.0):
                        tokens[r, i] = x
                        continue
                    rest = [max(p[t] - q.get(t, 0.0), 0.0) for t in ids]
                    w = rest if sum(rest) > 0 else [p[t] for t in ids]
                else:
                    w = [p[t] for t in ids]
                w = torch.tensor(w, dtype=F64)
            else:
                z = s['logits'][r * (T + 1) + i].double() / case['temperature']
                p = torch.exp(z - torch.logsumexp(z, 0))
                ids = None
                if i < T:
                    x = int(s['drafts'][r, i])
                    if case['probs']:
                        q = s['q'][r * T + i].double()
                    else:
                        q = torch.zeros_like(p)
                        q[x] = 1.0
                    if float(s['uniform'][r, i]) * float(q[x]) < float(p[x]):
                        tokens[r, i] = x
                        continue
                    rest = torch.relu(p - q)
                    w = rest if float(rest.sum()) > 0 else p
                else:
                    w = p
            c = torch.cumsum(w, 0)
            j = int(torch.searchsorted(c, float(s['uniform'][r, T]) * float(c[-1]), right=True))
            tokens[r, i], count[r] = (j if ids is None else ids[j]), i + 1
            break
    return tokens, count
