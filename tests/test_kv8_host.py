"""The 8-bit KV cache and token scoring without a GPU: the oracle's numbers,
plans, the refusals of the C ABI and of the Python entry points, and which
launches a pool takes."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from aios_amd import _lib, paged
from aios_amd.attention import backend as bk
from aios_amd.attention.backend import Mi355xAttentionBackend, Mi355xAttentionMetadata
from aios_amd.ime import CandidateGroupEngine, CandidateGroupRuntime, ScoredContinuation
from aios_amd.kernel import store_cache8
from aios_amd.kvcache import MHAKVCache, MHAKVCache8
from aios_amd.layers import HipOps
from aios_amd.sample import token_logprobs
from oracle import kv8 as okv8

FP8 = torch.float8_e4m3fn
BF16 = torch.bfloat16


# -- the oracle ---------------------------------------------------------------

def test_oracle_rounds_as_torch_does():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.linspace(-0.02, 0.02, 20001)])
    x = torch.cat([x, torch.arange(256, dtype=torch.uint8).view(FP8).float().nan_to_num(0.0)])
    want = x.to(FP8).double().numpy()
    assert (okv8.round_e4m3(x.double().numpy()) == want).all()


def test_oracle_scales_are_the_smallest_that_fit():
    x = np.array([[448.0, 1], [448.01, 1], [0, 0], [2.0 ** -130, 0], [3e38, -3.3e38], [1, np.nan]])
    codes, s = okv8.quantize_rows(x)
    assert s[0] == 1 and s[1] == 2 and s[2] == 2.0 ** -110 and s[3] == 2.0 ** -110
    assert np.isnan(s[5]) and codes[5, 1] == 0
    for c, k, row in zip(codes[:2], s[:2], x[:2]):
        assert np.abs(c).max() <= 448 and np.abs(c * k - row).max() <= 2.0 ** -4 * np.abs(row).max()


# -- plans ---------------------------------------------------------------------

def _plan8(phase, cu_q, cu_k, hq=32, hkv=8, d=128, shared=0, ws=1 << 30, chunk=0, split=0, page=1):
    cu_q, cu_k = (np.asarray(c, dtype=np.int32) for c in (cu_q, cu_k))
    p = _lib.AttnPlan()
    rc = _lib.lib().aios_attn_plan8(phase, cu_q.ctypes.data, cu_k.ctypes.data, len(cu_q) - 1, hq, hkv,
                                    d, page, shared, ws, chunk, split, p)
    return rc, p


def _decode8(lens, **kw):
    return _plan8(_lib.PHASE_DECODE, np.arange(len(lens) + 1), np.cumsum([0, *lens]), **kw)


def test_plan_refusals():
    bad = _lib.PHASE_DECODE8
    assert _plan8(bad, [0, 1], [0, 5])[0] == _lib.AIOS_ERR_INVALID
    assert _decode8([5], page=16)[0] == _lib.AIOS_ERR_UNSUPPORTED
    assert _decode8([5], hq=12, hkv=8)[0] == _lib.AIOS_ERR_INVALID
    assert _decode8([5], d=80)[0] == _lib.AIOS_ERR_UNSUPPORTED
    assert _decode8([5], hq=40, hkv=8)[0] == _lib.AIOS_ERR_UNSUPPORTED
    assert _decode8([5, 3], shared=4)[0] == _lib.AIOS_ERR_INVALID
    assert _decode8([5], shared=-1)[0] == _lib.AIOS_ERR_INVALID
    assert _decode8([0, 3])[0] == _lib.AIOS_ERR_INVALID
    assert _plan8(_lib.PHASE_DECODE, [0, 2], [0, 5])[0] == _lib.AIOS_ERR_INVALID
    assert _plan8(_lib.PHASE_PREFILL, [0, 6], [0, 5])[0] == _lib.AIOS_ERR_INVALID
    assert _plan8(_lib.PHASE_PREFILL, [1, 6], [0, 9])[0] == _lib.AIOS_ERR_INVALID
    assert _decode8([9000] * 4, ws=1024)[0] == _lib.AIOS_ERR_WORKSPACE
    with pytest.raises(ValueError):
        paged.plan("decode", [0, 1], [0, 5], 8, 2, 64, kv_bits=4)


def test_plans_cover_every_position():
    """Over random batches: parts a row may have are within the combine's
    bound, every row's parts cover it, and the workspace holds every part."""
    rng = np.random.default_rng(5)
    for _ in range(400):
        batch = int(rng.integers(1, 70))
        top = int(2 ** rng.uniform(0, 17))
        lens = rng.integers(1, top + 1, batch)
        g, hkv, d = int(rng.choice([1, 2, 3, 4, 6, 8])), int(rng.integers(1, 17)), int(rng.choice([64, 96, 128]))
        shared = int(rng.integers(0, lens.min() + 1)) if rng.random() < 0.5 else 0
        split = int(rng.integers(1, top + 200)) if rng.random() < 0.3 else 0
        chunk = int(rng.integers(1, 300)) if rng.random() < 0.3 else 0
        rc, p = _decode8(lens, hq=g * hkv, hkv=hkv, d=d, shared=shared, split=split, chunk=chunk,
                         ws=1 << 40)
        assert rc == 0
        own = lens - p.prefix_len
        assert 1 <= p.num_parts <= 64  # a lane of the combine for each
        if p.prefix_len:
            assert p.prefix_len == shared
            assert p.num_prefix_chunks * p.prefix_chunk_len >= p.prefix_len
            assert (p.num_prefix_chunks - 1) * p.prefix_chunk_len < p.prefix_len
        else:
            assert p.num_prefix_chunks == 0
        if p.suffix_parts_per_item == 0:  # equal parts of long rows
            parts = -(-own // p.suffix_split_len)
            assert p.num_suffix_splits == parts.sum()
            assert p.num_prefix_chunks + parts.max() <= p.num_parts
        else:
            assert p.num_parts == p.num_prefix_chunks + p.suffix_parts_per_item
        if p.num_parts > 1:
            states = batch * hkv * p.num_parts * g
            assert p.ws_parts_lse >= states * d * 2 and p.ws_bytes >= p.ws_parts_lse + states * 8


def test_plans_of_the_largest_parameters():
    top = 2 ** 31 - 1
    rc, p = _decode8([400] * 8, shared=400, chunk=top, split=top)
    assert rc == 0 and p.num_prefix_chunks == 1 and p.prefix_chunk_len >= 400
    rc, p = _decode8([top // 4] * 4, split=1, ws=1 << 50)
    assert rc == 0 and p.num_parts <= 64 and p.suffix_split_len * 64 >= top // 4
    rc, p = _plan8(_lib.PHASE_PREFILL, np.arange(5), np.arange(5) * (top // 4), ws=1 << 50)
    assert rc == 0 and p.num_parts >= 1


def test_prefill_plans_of_few_rows():
    """Parts cover every tile; without room for states the KV range stays whole."""
    rng = np.random.default_rng(7)
    for _ in range(300):
        batch = int(rng.integers(1, 80))
        g, hkv, d = int(rng.choice([1, 2, 3, 4, 6, 8])), int(rng.integers(1, 17)), int(rng.choice([64, 96, 128]))
        new = rng.integers(0, 64 // g + 1, batch)
        kv = new + rng.integers(0, int(2 ** rng.uniform(0, 15)) + 1, batch)
        cu_q, cu_k = np.cumsum([0, *new]), np.cumsum([0, *kv])
        for room in (1 << 40, 0):
            rc, p = _plan8(_lib.PHASE_PREFILL, cu_q, cu_k, hq=g * hkv, hkv=hkv, d=d, ws=room)
            assert rc == 0
            rows = min(int(new.max()), 128 // g) * g
            if p.num_parts:
                assert p.num_parts * p.prefix_chunk_len >= kv.max() and p.prefix_chunk_len % 32 == 0
            if p.num_parts > 1:
                parts = batch * hkv * p.num_q_tiles * p.num_parts
                assert p.ws_parts_lse >= parts * rows * d * 4
                assert p.ws_bytes >= p.ws_parts_lse + parts * rows * 8
            else:
                assert p.ws_bytes == 0
            assert p.ws_bytes <= room


# -- the C ABI refuses before it launches ---------------------------------------

ADDR = 1 << 20  # an aligned address that no refused call reads


def _append(k8=ADDR, v8=ADDR, s=ADDR, pages=8, hkv=2, d=64, loc=ADDR, k=ADDR, ks=128, v=ADDR, vs=128,
            n=3):
    return _lib.lib().aios_kv8_append(k8, v8, s, pages, hkv, d, loc, k, ks, v, vs, n, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(k8=None), "INVALID"), (dict(v8=None), "INVALID"), (dict(s=None), "INVALID"),
    (dict(loc=None), "INVALID"), (dict(k=None), "INVALID"), (dict(v=None), "INVALID"),
    (dict(n=-1), "INVALID"), (dict(pages=-1), "INVALID"), (dict(hkv=0), "INVALID"),
    (dict(d=80), "UNSUPPORTED"), (dict(k8=ADDR + 8), "INVALID"), (dict(v8=ADDR + 8), "INVALID"),
    (dict(s=ADDR + 2), "INVALID"), (dict(pages=1 << 24), "UNSUPPORTED"),
    (dict(pages=(1 << 24) - 1, hkv=8), "UNSUPPORTED"),
    (dict(ks=126), "INVALID"), (dict(vs=129), "INVALID"), (dict(k=ADDR + 2), "INVALID"),
    (dict(v=ADDR + 2), "INVALID"), (dict(n=1 << 40), "UNSUPPORTED")])
def test_append_refuses(kw, rc):
    assert _append(**kw) == getattr(_lib, "AIOS_ERR_" + rc)


def test_an_empty_append_launches_nothing():
    assert _append(n=0) == 0


def _rope_append(qkv=ADDR, stride=512, n=3, hq=4, hkv=2, d=64, qw=ADDR, kw=ADDR, cos=ADDR, sin=ADDR,
                 rows=16, pos=ADDR, q=ADDR, k8=ADDR, v8=ADDR, s=ADDR, pages=8, loc=ADDR):
    return _lib.lib().aios_qk_norm_rope_append8(qkv, stride, n, hq, hkv, d, qw, kw, cos, sin, rows, pos,
                                                q, k8, v8, s, pages, loc, 1e-6, None)


@pytest.mark.parametrize("kw", [
    dict(qkv=None), dict(qw=None), dict(kw=None), dict(cos=None), dict(sin=None), dict(pos=None),
    dict(q=None), dict(loc=None), dict(n=-1), dict(hq=0), dict(hkv=0), dict(rows=0), dict(stride=511),
    dict(stride=510), dict(qkv=ADDR + 2), dict(q=ADDR + 2), dict(k8=ADDR + 4), dict(s=None)])
def test_rope_append_refuses(kw):
    assert _rope_append(**kw) == _lib.AIOS_ERR_INVALID


def _attn(p, scale=0.1, q=ADDR, qs=None, k8=ADDR, v8=ADDR, s=ADDR, pages=64, idx=ADDR, cu_q=ADDR, cu_k=ADDR,
          out=ADDR, ws=ADDR, ws_bytes=1 << 40, new=None):
    lib, qs = _lib.lib(), p.num_qo_heads * p.head_dim if qs is None else qs
    if p.phase in (_lib.PHASE_PREFILL8, _lib.PHASE_PREFILL):
        return lib.aios_attn_prefill8(p, q, qs, k8, v8, s, pages, idx, cu_q, cu_k, out, ws, ws_bytes,
                                      scale, None)
    if new is None:
        return lib.aios_attn_decode8(p, q, qs, k8, v8, s, pages, idx, cu_k, out, ws, ws_bytes, scale,
                                     None)
    k, ks, v, vs, loc = new
    return lib.aios_attn_append_decode8(p, q, qs, k, ks, v, vs, loc, k8, v8, s, pages, idx, cu_k, out,
                                        ws, ws_bytes, scale, None)


BAD_ATTN = [dict(q=None), dict(k8=None), dict(v8=None), dict(s=None), dict(idx=None), dict(cu_k=None),
            dict(out=None), dict(qs=4088), dict(qs=4100), dict(q=ADDR + 8), dict(out=ADDR + 8),
            dict(k8=ADDR + 8), dict(s=ADDR + 2), dict(pages=-1), dict(scale=0.0), dict(scale=-0.1),
            dict(scale=float("nan")), dict(scale=float("inf"))]


@pytest.mark.parametrize("kw", BAD_ATTN + [dict(ws=ADDR + 16), dict(ws=None), dict(ws_bytes=16)])
def test_decode_refuses(kw):
    rc, p = _decode8([9000] * 4)
    assert rc == 0 and p.ws_bytes > 0
    short = "ws" in kw and kw["ws"] is None or "ws_bytes" in kw
    assert _attn(p, **kw) == (_lib.AIOS_ERR_WORKSPACE if short else _lib.AIOS_ERR_INVALID)


@pytest.mark.parametrize("kw", BAD_ATTN + [dict(cu_q=None)])
def test_prefill_refuses(kw):
    rc, p = _plan8(_lib.PHASE_PREFILL, [0, 5, 9], [0, 30, 40])
    assert rc == 0
    assert _attn(p, **kw) == _lib.AIOS_ERR_INVALID


NEW = [ADDR, 1024, ADDR, 1024, ADDR]


@pytest.mark.parametrize("at,bad", [(0, None), (2, None), (4, None), (1, 1022), (3, 1025), (0, ADDR + 2),
                                    (2, ADDR + 2)])
def test_append_decode_refuses(at, bad):
    _, p = _decode8([40] * 4)
    new = list(NEW)
    new[at] = bad
    assert _attn(p, new=new) == _lib.AIOS_ERR_INVALID


def test_append_decode_needs_a_position_behind_the_prefix():
    rc, p = _decode8([400] * 8, shared=400)
    assert rc == 0 and p.prefix_len == 400
    assert _attn(p, new=NEW) == _lib.AIOS_ERR_INVALID


def test_a_plan_of_another_phase_or_cache_is_refused():
    lib = _lib.lib()
    _, p8 = _decode8([40] * 4)
    _, f8 = _plan8(_lib.PHASE_PREFILL, [0, 5], [0, 30])
    cu = np.arange(5, dtype=np.int32)
    p = _lib.AttnPlan()
    assert lib.aios_attn_plan(_lib.PHASE_DECODE, cu.ctypes.data, (cu * 40).ctypes.data, 4, 32, 8, 128, 1,
                              0, 1 << 30, 0, 0, p) == 0
    dec = (ADDR, 4096, ADDR, ADDR, ADDR, 64, ADDR, ADDR, ADDR, ADDR, 1 << 40, 0.1, None)
    assert lib.aios_attn_decode8(p, *dec) == _lib.AIOS_ERR_INVALID
    assert lib.aios_attn_decode8(f8, *dec) == _lib.AIOS_ERR_INVALID
    pre = (ADDR, 4096, ADDR, ADDR, ADDR, 64, ADDR, ADDR, ADDR, ADDR, ADDR, 1 << 40, 0.1, None)
    assert lib.aios_attn_prefill8(p8, *pre) == _lib.AIOS_ERR_INVALID
    bf16 = (ADDR, 4096, ADDR, ADDR, 64, ADDR, ADDR, ADDR, ADDR, 1 << 40, 0.1, None)
    assert lib.aios_attn_decode(p8, *bf16) == _lib.AIOS_ERR_INVALID


def test_token_logprobs_c_refusals():
    lib = _lib.lib()

    def call(x=ADDR, stride=100, rows=3, vocab=100, size=2, tok=ADDR, top=2, lp=ADDR, ent=ADDR, ids=ADDR,
             alt=ADDR):
        return lib.aios_token_logprobs(x, stride, rows, vocab, size, tok, top, lp, ent, ids, alt, None, 0,
                                       None)

    for kw in (dict(x=None), dict(tok=None), dict(lp=None), dict(ent=None), dict(ids=None),
               dict(alt=None), dict(rows=-1), dict(vocab=0), dict(stride=99), dict(stride=-1),
               dict(top=-1), dict(vocab=20, top=21), dict(x=ADDR + 1), dict(x=ADDR + 2, size=4)):
        assert call(**kw) == _lib.AIOS_ERR_INVALID, kw
    for kw in (dict(size=1), dict(top=33), dict(rows=(1 << 24) + 1),
               dict(vocab=(1 << 30) + 1, stride=0)):
        assert call(**kw) == _lib.AIOS_ERR_UNSUPPORTED, kw
    assert call(rows=0) == 0


def test_token_logprobs_workspace():
    ws = _lib.lib().aios_token_logprobs_workspace
    assert ws(0, 100, 0) == 0 and ws(5, 0, 0) == 0 and ws(-1, 100, 5) == 0
    assert ws(1, 151936, 0) > 0


# -- Python entry points ---------------------------------------------------------

class Gpu(torch.Tensor):
    """A CPU tensor that says it is on GPU 0."""

    is_cuda = True

    def get_device(self):
        return getattr(self, "on", 0)


def _gpu(*shape, dtype=BF16, on=0):
    t = torch.zeros(*shape, dtype=dtype).as_subclass(Gpu)
    t.on = on
    return t


class _Reached(Exception):
    pass


@pytest.fixture
def no_launch(monkeypatch):
    """Every C call raises: refusals come before any."""
    real = _lib.lib()

    class Lib:
        def __getattr__(self, name):
            if name in ("aios_attn_plan8", "aios_attn_plan", "aios_last_error"):
                return getattr(real, name)

            def fn(*a):
                raise _Reached(name)
            return fn

    monkeypatch.setattr(_lib, "lib", Lib)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 0, raising=False)


def _store_args(**kw):
    a = dict(k8=_gpu(8, 2, 64, dtype=FP8), v8=_gpu(8, 2, 64, dtype=FP8), scales=_gpu(2, 8, 2),
             indices=_gpu(3, dtype=torch.int32), k=_gpu(3, 2, 64), v=_gpu(3, 2, 64))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    {}, dict(k=_gpu(3, 6, 64)[:, 2:4], v=_gpu(3, 6, 64)[:, 4:]), dict(indices=_gpu(3, dtype=torch.int64))])
def test_store_launches(no_launch, kw):
    with pytest.raises(_Reached, match="aios_kv8_append"):
        store_cache8(**_store_args(**kw))


@pytest.mark.parametrize("kw", [
    dict(k8=_gpu(8, 2, 64)), dict(v8=_gpu(8, 2, 64, dtype=torch.float8_e5m2)), dict(k8=_gpu(8, 128, dtype=FP8)),
    dict(v8=_gpu(9, 2, 64, dtype=FP8)), dict(scales=_gpu(8, 2, 2)), dict(scales=_gpu(2, 8, 2, dtype=torch.float32)),
    dict(scales=_gpu(2, 2, 8).transpose(1, 2)), dict(indices=_gpu(4, dtype=torch.int32)),
    dict(k=_gpu(3, 2, 64, dtype=torch.float16)), dict(v=_gpu(3, 2, 64, dtype=torch.float32)),
    dict(k=_gpu(3, 3, 64)), dict(v=_gpu(2, 2, 64)), dict(k=_gpu(3, 64, 2).transpose(1, 2)),
    dict(k=_gpu(3, 4, 64)[:, ::2]), dict(indices=_gpu(3, dtype=torch.float32)),
    dict(indices=_gpu(3, dtype=torch.bool)), dict(k8=_gpu(8, 2, 128, dtype=FP8)[..., :64]),
    dict(scales=_gpu(2, 8, 2, on=1)), dict(indices=_gpu(3, dtype=torch.int32, on=1)),
    dict(k=torch.zeros(3, 2, 64, dtype=BF16))])
def test_store_refuses(no_launch, kw):
    with pytest.raises(ValueError):
        store_cache8(**_store_args(**kw))


def _decode_args(**kw):
    a = dict(p=paged.plan("decode", [0, 1, 2, 3], [0, 9, 15, 22], 8, 2, 64, kv_bits=8), q=_gpu(3, 8, 64),
             k8=_gpu(30, 2, 64, dtype=FP8), v8=_gpu(30, 2, 64, dtype=FP8), scales=_gpu(2, 30, 2),
             indices=_gpu(22, dtype=torch.int32), cu_k=_gpu(4, dtype=torch.int32))
    a.update(kw)
    return a


BAD_CACHE = [dict(k8=_gpu(30, 2, 64)), dict(v8=_gpu(29, 2, 64, dtype=FP8)), dict(scales=_gpu(30, 2, 2)),
             dict(k8=_gpu(30, 4, 64, dtype=FP8)[:, :2]), dict(scales=_gpu(2, 30, 2, on=1)),
             dict(k8=_gpu(30, 4, 64, dtype=FP8), v8=_gpu(30, 4, 64, dtype=FP8)),
             dict(indices=_gpu(21, dtype=torch.int32)), dict(cu_k=_gpu(4, dtype=torch.int64)),
             dict(indices=_gpu(44, dtype=torch.int32)[::2]), dict(cu_k=_gpu(4, dtype=torch.int32, on=1)),
             dict(q=_gpu(3, 8, 64, dtype=torch.float16)), dict(q=_gpu(3, 8, 32)), dict(q=_gpu(3, 6, 64)),
             dict(q=_gpu(3, 64, 8).transpose(1, 2)), dict(q=torch.zeros(3, 8, 64, dtype=BF16)),
             dict(out=_gpu(2, 8, 64)), dict(out=_gpu(3, 8, 64, dtype=torch.float32)),
             dict(out=_gpu(3, 8, 128)[..., :64])]


@pytest.mark.parametrize("kw", BAD_CACHE + [dict(q=_gpu(2, 8, 64)),
                                            dict(workspace=torch.empty(99, dtype=torch.uint8))])
def test_decode_entry_refuses(no_launch, kw):
    with pytest.raises(_Reached, match="aios_attn_decode8"):
        paged.decode8(**_decode_args())
    with pytest.raises(ValueError):
        paged.decode8(**_decode_args(**kw))


def test_decode_entry_needs_its_workspace_and_plan(no_launch):
    p = paged.plan("decode", [0, 1], [0, 40000], 8, 2, 64, kv_bits=8)
    kw = dict(q=_gpu(1, 8, 64), indices=_gpu(40000, dtype=torch.int32), cu_k=_gpu(2, dtype=torch.int32))
    assert p.ws_bytes > 0
    with pytest.raises(RuntimeError, match="workspace"):
        paged.decode8(**_decode_args(p=p, **kw))
    with pytest.raises(ValueError, match="8-bit"):
        paged.decode8(**_decode_args(p=paged.plan("decode", [0, 1, 2, 3], [0, 9, 15, 22], 8, 2, 64)))
    with pytest.raises(ValueError):
        paged.decode(_decode_args()["p"], _gpu(3, 8, 64), _gpu(30, 2, 64), _gpu(30, 2, 64),
                     _gpu(22, dtype=torch.int32), _gpu(4, dtype=torch.int32))


@pytest.mark.parametrize("kw", [
    dict(k=_gpu(3, 2, 64, dtype=torch.float16)), dict(v=_gpu(3, 3, 64)), dict(k=_gpu(2, 2, 64)),
    dict(v=_gpu(3, 2, 128)[..., ::2]), dict(k=_gpu(3, 2, 64, on=1)), dict(out_loc=_gpu(2, dtype=torch.int32)),
    dict(out_loc=_gpu(3, dtype=torch.int64)), dict(out_loc=torch.zeros(3, dtype=torch.int32))])
def test_append_decode_entry_refuses(no_launch, kw):
    a = _decode_args(k=_gpu(3, 2, 64), v=_gpu(3, 2, 64), out_loc=_gpu(3, dtype=torch.int32))
    with pytest.raises(_Reached, match="aios_attn_append_decode8"):
        paged.append_decode8(**a)
    with pytest.raises(ValueError):
        paged.append_decode8(**{**a, **kw})


@pytest.mark.parametrize("kw", [
    dict(q_norm=_gpu(32)), dict(k_norm=_gpu(64, dtype=torch.float32)), dict(cos=_gpu(40, 32)),
    dict(sin=_gpu(41, 64)), dict(cos=_gpu(40, 64, dtype=torch.float32)), dict(cos=_gpu(64, 40).T),
    dict(positions=_gpu(2, dtype=torch.int32)), dict(positions=_gpu(3, dtype=torch.int64)),
    dict(q_norm=_gpu(64, on=1)), dict(sin=_gpu(40, 64, on=1))])
def test_append_decode_rope_entry_refuses(no_launch, kw):
    a = _decode_args(k=_gpu(3, 2, 64), v=_gpu(3, 2, 64), out_loc=_gpu(3, dtype=torch.int32),
                     q_norm=_gpu(64), k_norm=_gpu(64), cos=_gpu(40, 64), sin=_gpu(40, 64),
                     positions=_gpu(3, dtype=torch.int32), eps=1e-6)
    with pytest.raises(_Reached, match="aios_attn_append_decode_rope8"):
        paged.append_decode_rope8(**a)
    with pytest.raises(ValueError):
        paged.append_decode_rope8(**{**a, **kw})


@pytest.mark.parametrize("kw", BAD_CACHE + [dict(cu_q=_gpu(3, dtype=torch.int32))])
def test_prefill_entry_refuses(no_launch, kw):
    a = _decode_args(p=paged.plan("prefill", [0, 1, 2, 3], [0, 9, 15, 22], 8, 2, 64, kv_bits=8),
                     cu_q=_gpu(4, dtype=torch.int32))
    with pytest.raises(_Reached, match="aios_attn_prefill8"):
        paged.prefill8(**a)
    with pytest.raises(ValueError):
        paged.prefill8(**{**a, **kw})
    with pytest.raises(RuntimeError, match="flat Q"):
        paged.prefill8(**{**a, "q": _gpu(4, 8, 64)})


def test_another_device_than_the_current_one_is_refused(no_launch, monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    with pytest.raises(ValueError, match="current device"):
        store_cache8(**_store_args())
    with pytest.raises(ValueError, match="current device"):
        paged.decode8(**_decode_args())


@pytest.mark.parametrize("kw", [
    dict(qkv=_gpu(3, 520)), dict(qkv=_gpu(3, 512, dtype=torch.float16)), dict(q_weight=_gpu(32)),
    dict(k_weight=_gpu(64, dtype=torch.float32)), dict(cos=_gpu(16, 64)),
    dict(positions=_gpu(3, dtype=torch.int64)), dict(k8=_gpu(8, 2, 64)), dict(scales=_gpu(8, 2, 2)),
    dict(v8=_gpu(9, 2, 64, dtype=FP8)), dict(out_loc=_gpu(2, dtype=torch.int32)),
    dict(out_loc=torch.zeros(3, dtype=torch.int32)), dict(scales=_gpu(2, 8, 2, on=1))])
def test_rope_append_entry_refuses(no_launch, kw):
    f32 = torch.float32
    a = dict(qkv=_gpu(3, 512), q_weight=_gpu(64), k_weight=_gpu(64), cos=_gpu(16, 64, dtype=f32),
             sin=_gpu(16, 64, dtype=f32), positions=_gpu(3, dtype=torch.int32), num_qo_heads=4, eps=1e-6,
             k8=_gpu(8, 2, 64, dtype=FP8), v8=_gpu(8, 2, 64, dtype=FP8), scales=_gpu(2, 8, 2),
             out_loc=_gpu(3, dtype=torch.int32))
    with pytest.raises(ValueError):
        HipOps.qk_norm_rope_append8(**{**a, **kw})


@pytest.mark.parametrize("logits,tokens,top", [
    (_gpu(3, 50, dtype=torch.float16), _gpu(3, dtype=torch.int64), 0),
    (_gpu(150), _gpu(3, dtype=torch.int64), 0),
    (_gpu(3, 100)[:, ::2], _gpu(3, dtype=torch.int64), 0),
    (torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64), 0),
    (_gpu(3, 50), _gpu(3, dtype=torch.int32), 0), (_gpu(3, 50), _gpu(4, dtype=torch.int64), 0),
    (_gpu(3, 50), _gpu(3, dtype=torch.int64, on=1), 0), (_gpu(3, 50), _gpu(3, dtype=torch.int64), -1),
    (_gpu(3, 50), _gpu(3, dtype=torch.int64), 33), (_gpu(3, 20), _gpu(3, dtype=torch.int64), 21)])
def test_token_logprobs_refuses(no_launch, logits, tokens, top):
    with pytest.raises(ValueError):
        token_logprobs(logits, tokens, top)


# -- the pool and the backend ------------------------------------------------------

@pytest.mark.parametrize("kw", [dict(dtype=BF16), dict(head_dim=80)])
def test_pool_refuses(kw):
    a = dict(num_kv_heads=2, num_layers=1, head_dim=64, num_pages=8, page_size=1, dtype=FP8, device="cuda")
    with pytest.raises(ValueError):
        MHAKVCache8(**{**a, **kw})
    with pytest.raises(AssertionError):
        MHAKVCache8(**{**a, "device": "cpu"})
    with pytest.raises(AssertionError):
        MHAKVCache8(**{**a, "page_size": 16})


def _pool(cls=MHAKVCache8, heads=2):
    p = cls.__new__(cls)
    p._kv_buffer = torch.empty(2, 2, 8, 1, heads, 64, dtype=FP8)
    p._k_buffer, p._v_buffer = p._kv_buffer
    p._scales = torch.zeros(2, heads, 8, 2, dtype=BF16)
    p._num_layers, p._device = 2, torch.device("cuda")
    p._storage_shape = (8, heads, 64)
    return p


def test_pool_views():
    p = _pool()
    k8, v8, s = p.layer(1)
    assert k8.shape == v8.shape == (8, 2, 64) and s.shape == (2, 8, 2)
    assert k8.data_ptr() == p.k_cache(1).data_ptr() and v8.data_ptr() == p.v_cache(1).data_ptr()
    assert s.data_ptr() == p.scales(1).data_ptr() != p.scales(0).data_ptr()
    assert (p.num_pages, p.num_layers, p.dtype, p.row_shape) == (8, 2, FP8, (2, 64))
    assert bk._kv_bits(p) == 8 and bk._kv_bits(None) == 16
    assert bk._kv_bits(SimpleNamespace(dtype=BF16, layer=None)) == 16


class _OwnStore(MHAKVCache8):
    def store_kv(self, k, v, out_loc, layer_id):
        return super().store_kv(k, v, out_loc, layer_id)


class _OwnLayer(MHAKVCache8):
    def layer(self, index):
        return super().layer(index)


class _Plain(MHAKVCache8):
    pass


def _batch(loc=None, tokens=3, phase="prefill", total_q=3):
    md = object.__new__(Mi355xAttentionMetadata)
    md.plan = _lib.AttnPlan()
    md.plan.total_q = total_q
    loc = _gpu(tokens, dtype=torch.int32) if loc is None else loc
    return SimpleNamespace(is_prefill=phase == "prefill", is_decode=phase != "prefill", out_loc=loc,
                           attn_metadata=md, fused_append=False)


def test_which_prefills_write_in_the_rotating_launch():
    be = Mi355xAttentionBackend(SimpleNamespace(num_qo_heads=4, num_kv_heads=2, head_dim=64))
    qkv = torch.zeros(3, 512, dtype=BF16)
    assert be.append_rope8_applies(qkv, _pool(), _batch())
    assert be.append_rope8_applies(qkv, _pool(_Plain), _batch())
    assert not be.append_rope_applies(qkv, _pool(), _batch())  # (the bfloat16 launch)
    for pool in (_pool(_OwnStore), _pool(_OwnLayer), _pool(heads=3)):
        assert not be.append_rope8_applies(qkv, pool, _batch())
    own = _pool()
    own.store_kv = lambda *a: None
    assert not be.append_rope8_applies(qkv, own, _batch())
    bf16 = MHAKVCache.__new__(MHAKVCache)
    bf16._kv_buffer, bf16._storage_shape = torch.empty(2, 1, 8, 1, 2, 64, dtype=BF16), (8, 2, 64)
    assert not be.append_rope8_applies(qkv, bf16, _batch())
    assert be.append_rope_applies(qkv, bf16, _batch())
    for b in (_batch(phase="decode"), _batch(tokens=2), _batch(total_q=4),
              _batch(loc=_gpu(3, dtype=torch.int64)), _batch(loc=_gpu(6, dtype=torch.int32)[::2])):
        assert not be.append_rope8_applies(qkv, _pool(), b)
    assert not be.append_rope8_applies(qkv.float(), _pool(), _batch())


# -- scoring ------------------------------------------------------------------------

def _engine():
    rt = object.__new__(CandidateGroupRuntime)
    rt.config = SimpleNamespace(max_position_embeddings=64)
    rt.max_context, rt.num_pages, rt.max_attempts = 48, 40, 2
    rt.model = SimpleNamespace(w={"embed": torch.zeros(100, 4)})
    return CandidateGroupEngine(rt, use_graphs=False)


@pytest.mark.parametrize("prefix,conts,top", [
    ([], [[1]], 0), ([1, 2], [[3], []], 0), ([1, 100], [[3]], 0), ([1, -1], [[3]], 0),
    ([1], [[100]], 0), ([1], [[3, -1]], 0), ([1], [[3]], -1), ([1], [[3]], 33),
    ([1] * 40, [[2] * 10], 0), ([1] * 30, [[2] * 6, [2] * 7], 0)])
def test_score_refuses(prefix, conts, top):
    eng = _engine()
    eng._prepare_prefix = lambda *a: pytest.fail("refused calls prepare nothing")
    with pytest.raises(ValueError):
        eng.score(prefix, conts, top)


def test_runtime_refuses_other_widths():
    with pytest.raises(ValueError, match="kv_bits"):
        CandidateGroupRuntime(None, {}, kv_bits=4)


def test_scored_continuation_average():
    s = ScoredContinuation((1, 2), (-1.0, -3.0), (0.5, 0.5))
    assert s.average_logprob == -2.0 and s.alternatives == ()


def test_error_texts_reach_python():
    assert _append(k8=None) == _lib.AIOS_ERR_INVALID
    assert b"kv8_append" in _lib.lib().aios_last_error()
    assert isinstance(ctypes.c_char_p(_lib.lib().aios_last_error()).value, bytes)
