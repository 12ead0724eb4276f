"""CPU: what the packed-prompt, shared-prefix and draft-verification entry points refuse before anything is launched, and the calls with
nothing to do (no device is needed for either)."""
import ctypes

import pytest

P16 = 0x10000                    # an aligned address that no refused call reads


@pytest.fixture(scope='module')
def L(built_lib):
    return built_lib


def refused(L, fn, d, word, **kw):
    for k, v in kw.items():
        assert hasattr(d, k), k
        setattr(d, k, v)
    assert fn(ctypes.byref(d), None) == -1, kw
    assert word.encode() in L.ifh_last_error(), (kw, L.ifh_last_error())


def rope():
    from infernos_amd._lib import RopePackedDesc
    d = RopePackedDesc()
    d.qkv = d.q_out = d.cos_sin = d.cache = d.cu = d.pos0 = P16
    d.qkv_ld, d.q_ld, d.cache_bs, d.cache_ts = 16 * 128, 16 * 128, 64 * 512, 512
    d.ntokens, d.nseqs, d.nheads, d.nkv, d.head_dim, d.max_pos, d.table_len = 5, 2, 12, 2, 128, 64, 64
    return d


@pytest.mark.parametrize('kw,word', [
    (dict(qkv=0), 'qkv'), (dict(cu=0), 'cu'), (dict(pos0=0), 'pos0'), (dict(cos_sin=0), 'cos_sin'), (dict(ntokens=-1), 'ntokens'),
    (dict(nseqs=-1), 'nseqs'), (dict(head_dim=24), 'head_dim'), (dict(qkv_ld=2040), 'qkv_ld'), (dict(qkv_ld=2049), 'qkv_ld'), (dict(q_ld=128), 'q_ld'),
    (dict(cache_ts=256), 'cache_ts'), (dict(cache_bs=63 * 512), 'cache_bs'), (dict(table_len=0), 'table_len'), (dict(max_pos=0), 'max_pos'),
    (dict(cache=P16 + 2), '15'), (dict(nkv=0), 'nkv')])
def test_rope_refusals(L, kw, word):
    refused(L, L.ifh_rope_append_packed_bf16, rope(), word, **kw)


def packed():
    from infernos_amd._lib import AttnPackedDesc
    d = AttnPackedDesc()
    d.q = d.cache = d.out = d.cu = d.key_len = P16
    d.q_ts, d.cache_bs, d.cache_ts, d.v_off, d.o_ts = 16 * 128, 64 * 512, 512, 256, 12 * 128
    d.ntokens, d.nseqs, d.nheads, d.nkv, d.head_dim, d.max_keys, d.scale = 5, 2, 12, 2, 128, 64, 0.1
    return d


def prefix():
    from infernos_amd._lib import AttnPrefixDesc
    d = AttnPrefixDesc()
    d.q = d.cache = d.out = d.prefix = d.key_len = d.ws = P16
    d.q_ts, d.prefix_ts, d.cache_bs, d.cache_ts, d.v_off, d.o_ts = 16 * 128, 512, 64 * 512, 512, 256, 12 * 128
    d.nrows, d.tokens_per_row, d.prefix_keys, d.nheads, d.nkv, d.head_dim, d.max_keys, d.scale = 5, 1, 100, 12, 2, 128, 64, 0.1
    d.ws_floats = 1 << 40
    return d


SHARED = [(dict(q=0), 'q'), (dict(out=0), 'out'), (dict(key_len=0), 'key_len'), (dict(head_dim=96), 'head_dim'), (dict(nheads=13), 'nheads'),
          (dict(nkv=0), 'nkv'), (dict(scale=0.0), 'scale'), (dict(scale=float('nan')), 'scale'), (dict(q_ts=1528), 'q_ts'), (dict(q_ts=2049), 'q_ts'),
          (dict(o_ts=1528), 'o_ts'), (dict(cache_ts=504), 'cache_ts'), (dict(v_off=-8), 'v_off'), (dict(v_off=257), 'v_off'), (dict(max_keys=0), 'max_keys'),
          (dict(max_keys=65), 'max_keys'), (dict(q=P16 + 8), '15'), (dict(ws=P16 + 4), '15')]


@pytest.mark.parametrize('kw,word', SHARED + [(dict(cu=0), 'cu'), (dict(ntokens=-1), 'ntokens'), (dict(nseqs=-2), 'nseqs'), (dict(ntokens=1 << 30), 'ntokens')])
def test_attn_packed_refusals(L, kw, word):
    refused(L, L.ifh_attn_packed_bf16, packed(), word, **kw)


@pytest.mark.parametrize('kw,word', SHARED + [(dict(prefix=0), 'prefix'), (dict(ws=0), 'ws'), (dict(nrows=-1), 'nrows'), (dict(tokens_per_row=0), 'tokens_per_row'),
                                              (dict(prefix_keys=0), 'prefix_keys'), (dict(prefix_ts=504), 'prefix_ts'), (dict(prefix_ts=516), 'prefix_ts'),
                                              (dict(prefix=P16 + 8), 'prefix'), (dict(ws_floats=10), 'ws_floats'), (dict(nrows=1 << 24), 'ntokens')])
def test_attn_prefix_refusals(L, kw, word):
    refused(L, L.ifh_attn_prefix_bf16, prefix(), word, **kw)


def verify():
    from infernos_amd._lib import VerifyDesc
    d = VerifyDesc()
    d.logits = d.drafts = d.uniform = d.out_tokens = d.out_count = d.ws = P16
    d.ld, d.q_ld, d.vocab, d.nrows, d.ndraft, d.temperature, d.ws_bytes = 1000, 1000, 1000, 4, 3, 1.0, 1 << 40
    return d


@pytest.mark.parametrize('kw,word', [
    (dict(logits=0), 'logits'), (dict(drafts=0), 'drafts'), (dict(uniform=0), 'uniform'), (dict(ws=0), 'ws'), (dict(out_count=0), 'out_count'),
    (dict(ld=999), 'ld'), (dict(draft_probs=P16, q_ld=999), 'q_ld'), (dict(vocab=0), 'vocab'), (dict(vocab=600000, ld=600000), 'vocab'), (dict(ndraft=64), 'ndraft'),
    (dict(ndraft=-1), 'ndraft'), (dict(nrows=-1), 'nrows'), (dict(nrows=40000), 'nrows'), (dict(temperature=-1.0), 'temperature'),
    (dict(temperature=float('nan')), 'temperature'), (dict(temperature=1e-9), 'temperature'), (dict(ws_bytes=64), 'ws_bytes'), (dict(ws=P16 + 8), 'ws')])
def test_verify_refusals(L, kw, word):
    refused(L, L.ifh_verify_drafts_f32, verify(), word, **kw)


def test_verify_topk_refusals(L):
    ok = dict(cand=P16, probs=P16, dc=P16, dp=P16, drafts=P16, lens=None, u=P16, nrows=2, ndraft=3, out=P16, cnt=P16)
    for kw, word in ((dict(cand=None), 'cand'), (dict(dp=None), 'draft_probs'), (dict(ndraft=64), 'ndraft'), (dict(nrows=-1), 'nrows'), (dict(drafts=None), 'drafts')):
        a = {**ok, **kw}
        assert L.ifh_verify_drafts_topk(*a.values(), None) == -1
        assert word.encode() in L.ifh_last_error()


def test_nothing_to_do(L):
    """no tokens, no sequences, no rows: accepted without a device"""
    for fn, d, k in ((L.ifh_rope_append_packed_bf16, rope(), 'ntokens'), (L.ifh_rope_append_packed_bf16, rope(), 'nseqs'),
                     (L.ifh_attn_packed_bf16, packed(), 'ntokens'), (L.ifh_attn_packed_bf16, packed(), 'nseqs'),
                     (L.ifh_attn_prefix_bf16, prefix(), 'nrows'), (L.ifh_verify_drafts_f32, verify(), 'nrows')):
        setattr(d, k, 0)
        assert fn(ctypes.byref(d), None) == 0
    assert L.ifh_attn_packed_ws_floats(0, 0, 12, 2, 128, 64) == 0 and L.ifh_verify_drafts_ws_bytes(0, 3) == 0
