"""What the operators over paged chunks and 8-bit caches refuse: the Python checks with every
launch replaced, and the C entries' own checks. No GPU is used."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mxflashattn_amd as mx
from mxflashattn_amd import native
from mxflashattn_amd.native import UnsupportedConfig

E4M3, INT8, BF16 = torch.float8_e4m3fn, torch.int8, torch.bfloat16


class Launched(Exception):
    pass


class NoLaunch:
    """The library, its launches replaced."""

    def __init__(self, lib):
        self._lib = lib

    def __getattr__(self, name):
        if not name.endswith("_launch") or name.endswith("per_launch"):
            return getattr(self._lib, name)

        def launch(*args):
            raise Launched(name)

        return launch


@pytest.fixture
def no_launch(monkeypatch):
    lib = NoLaunch(native.library())
    monkeypatch.setattr(native, "USE_TORCH_OP", False)
    monkeypatch.setattr(native, "library", lambda: lib)
    monkeypatch.setattr(native, "_require_device", lambda *t: t[0].device)
    monkeypatch.setattr(native, "_stream_handle", lambda device: 0)
    monkeypatch.setattr(native, "num_cus", lambda index: 256)
    monkeypatch.setattr(native, "_own_workspace", lambda device, stream, n: torch.empty(n))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def cache(dtype=BF16, pages=8, ps=16, hkv=2, hd=64):
    return torch.zeros(pages, ps, hkv, hd, dtype=dtype)


def scales(pages=8, hkv=2, ps=16, dtype=torch.float32):
    return torch.ones(pages, hkv, ps, dtype=dtype)


def prefill_args(codes=BF16, **change):
    a = dict(q=torch.zeros(10, 8, 64, dtype=BF16), k_cache=cache(codes), v_cache=cache(codes),
             cu_seqlens_q=ints(0, 4, 10), block_table=torch.zeros(2, 3, dtype=torch.int32),
             cache_seqlens=ints(4, 40), softmax_scale=0.1)
    if codes != BF16:
        a |= dict(k_scale=scales(), v_scale=scales())
    return a | change


def decode_args(codes=INT8, **change):
    a = dict(q=torch.zeros(2, 8, 64, dtype=BF16), k_cache=cache(codes), v_cache=cache(codes),
             block_table=torch.zeros(2, 3, dtype=torch.int32), cache_seqlens=ints(4, 40),
             softmax_scale=0.1, k_scale=scales(), v_scale=scales())
    return a | change


def write_args(codes=INT8, **change):
    a = dict(key=torch.zeros(5, 2, 64, dtype=BF16), value=torch.zeros(5, 2, 64, dtype=BF16),
             key_cache=cache(codes), value_cache=cache(codes), k_scale=scales(),
             v_scale=scales(), slot_mapping=torch.arange(5))
    return a | change


def gather_args(codes=INT8, **change):
    a = dict(key_cache=cache(codes), value_cache=cache(codes),
             block_table=torch.zeros(2, 3, dtype=torch.int32), cu_seqlens=ints(0, 4, 10),
             total=10, k_scale=scales(), v_scale=scales(), dtype=BF16)
    if codes == BF16:
        a |= dict(k_scale=None, v_scale=None)
    return a | change


def overlapping(*shape, dtype=BF16):
    return torch.zeros(1, dtype=dtype).expand(*shape)


BAD_ROW_SCALES = {
    "k missing": dict(k_scale=None),
    "v missing": dict(v_scale=None),
    "a number": dict(k_scale=0.5),
    "one value": dict(v_scale=torch.ones(1)),
    "64 bits": dict(v_scale=scales(dtype=torch.float64)),
    "pages": dict(k_scale=scales(pages=7)),
    "tokens before heads": dict(k_scale=torch.ones(8, 16, 2)),
    "tokens apart": dict(v_scale=torch.ones(8, 16, 2).transpose(1, 2)),
}
PREFILL = {
    "q of one token": dict(q=torch.zeros(8, 64, dtype=BF16)),
    "q in 32 bits": dict(q=torch.zeros(10, 8, 64)),
    "head dim of q": dict(q=torch.zeros(10, 8, 128, dtype=BF16)),
    "head dim 96": dict(q=torch.zeros(10, 8, 96, dtype=BF16), k_cache=cache(hd=96),
                        v_cache=cache(hd=96)),
    "heads": dict(q=torch.zeros(10, 7, 64, dtype=BF16)),
    "17 heads a kv head": dict(q=torch.zeros(10, 34, 64, dtype=BF16)),
    "cache of another type": dict(k_cache=cache(torch.float16), v_cache=cache(torch.float16)),
    "caches of two types": dict(v_cache=cache(E4M3)),
    "caches of two shapes": dict(v_cache=cache(pages=9)),
    "page size 12": dict(k_cache=cache(ps=12), v_cache=cache(ps=12)),
    "page size 8192": dict(k_cache=cache(pages=1, ps=8192), v_cache=cache(pages=1, ps=8192)),
    "caches of two layouts": dict(
        v_cache=torch.zeros(8, 2, 16, 64, dtype=BF16).transpose(1, 2)),
    "a strided last dim": dict(k_cache=torch.zeros(8, 16, 2, 128, dtype=BF16)[..., ::2],
                               v_cache=torch.zeros(8, 16, 2, 128, dtype=BF16)[..., ::2]),
    "offsets of one sequence": dict(cu_seqlens_q=ints(0, 10)),
    "offsets in two dims": dict(cu_seqlens_q=ints(0, 4, 10)[None]),
    "a table of one row": dict(block_table=torch.zeros(1, 3, dtype=torch.int32)),
    "a flat table": dict(block_table=ints(0, 1)),
    "a table without columns": dict(block_table=torch.zeros(2, 0, dtype=torch.int32)),
    "window -2": dict(window_left=-2),
    "cap -1": dict(softcap=-1.0),
    "cap inf": dict(softcap=float("inf")),
    "cap NaN": dict(softcap=float("nan")),
    "sinks of kv heads": dict(sinks=torch.zeros(2)),
    "slopes of kv heads": dict(alibi_slopes=torch.zeros(2)),
    "out of another shape": dict(out=torch.zeros(11, 8, 64, dtype=BF16)),
    "out of another type": dict(out=torch.zeros(10, 8, 64)),
    "out on itself": dict(out=overlapping(10, 1, 64).expand(10, 8, 64).clone()[:1].expand(
        10, 8, 64)),
    "out strided": dict(out=torch.zeros(10, 8, 128, dtype=BF16)[..., ::2]),
}


@pytest.mark.parametrize("codes", [BF16, E4M3, INT8])
def test_calls_within_the_contract_launch(no_launch, codes):
    with pytest.raises(Launched):
        mx.paged_prefill(**prefill_args(codes))
    with pytest.raises(Launched):
        mx.gather_cache(**gather_args(codes))
    if codes == BF16:
        return
    with pytest.raises(Launched):
        mx.paged_decode_split(**decode_args(codes))
    with pytest.raises(Launched):
        mx.quantize_and_cache(**write_args(codes))


@pytest.mark.parametrize("change", PREFILL.values(), ids=PREFILL)
def test_prefill(no_launch, change):
    with pytest.raises((ValueError, UnsupportedConfig)):
        mx.paged_prefill(**prefill_args(**change))


@pytest.mark.parametrize("codes", [E4M3, INT8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("change", BAD_ROW_SCALES.values(), ids=BAD_ROW_SCALES)
@pytest.mark.parametrize("call,args", [
    (mx.paged_prefill, prefill_args), (mx.paged_decode_split, decode_args),
    (mx.quantize_and_cache, write_args), (mx.gather_cache, gather_args),
], ids=["prefill", "decode", "write", "gather"])
def test_row_scales(no_launch, call, args, change, codes):
    with pytest.raises((ValueError, UnsupportedConfig)):
        call(**args(codes, **change))


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(2, 8, 96, dtype=BF16)),
    dict(q=torch.zeros(2, 5, 8, 64, dtype=BF16)),  # 20 columns, not causal
    dict(k_cache=cache(torch.uint8), v_cache=cache(torch.uint8)),
    dict(v_cache=cache(E4M3)),
    dict(cache_seqlens=ints(4)),
    dict(window_left=-2),
    dict(softcap=-1.0),
    dict(sinks=torch.zeros(2)),
    dict(out=torch.zeros(2, 8, 64)),
], ids=lambda c: "-".join(c))
def test_decode(no_launch, change):
    with pytest.raises((ValueError, UnsupportedConfig)):
        mx.paged_decode_split(**decode_args(**change))


@pytest.mark.parametrize("change", [
    dict(key=torch.zeros(5, 128, dtype=BF16)),
    dict(value=torch.zeros(4, 2, 64, dtype=BF16)),
    dict(key=torch.zeros(5, 2, 64), value=torch.zeros(5, 2, 64)),
    dict(key=torch.zeros(5, 2, 64, dtype=torch.float16)),
    dict(key_cache=cache(BF16), value_cache=cache(BF16)),
    dict(key_cache=cache(INT8, hkv=4), value_cache=cache(INT8, hkv=4)),
    dict(key_cache=cache(INT8)[0], value_cache=cache(INT8)[0]),
    dict(value_cache=torch.zeros(8, 2, 16, 64, dtype=INT8).transpose(1, 2)),
    dict(slot_mapping=torch.arange(4)),
    dict(slot_mapping=torch.arange(5)[None]),
    dict(key_cache=overlapping(8, 16, 2, 64, dtype=INT8),
         value_cache=overlapping(8, 16, 2, 64, dtype=INT8)),
    dict(k_scale=overlapping(8, 2, 1, dtype=torch.float32).expand(8, 2, 16)),
], ids=lambda c: "-".join(c))
def test_write(no_launch, change):
    with pytest.raises((ValueError, UnsupportedConfig)):
        mx.quantize_and_cache(**write_args(**change))


def test_write_of_k_over_v(no_launch):
    one, s = cache(INT8), scales()
    with pytest.raises(ValueError, match="share memory"):
        mx.quantize_and_cache(**write_args(key_cache=one, value_cache=one))
    with pytest.raises(ValueError, match="share memory"):
        mx.quantize_and_cache(**write_args(k_scale=s, v_scale=s))


@pytest.mark.parametrize("change", [
    dict(key_cache=cache(INT8)[0], value_cache=cache(INT8)[0]),
    dict(value_cache=cache(E4M3)),
    dict(value_cache=torch.zeros(8, 2, 16, 64, dtype=INT8).transpose(1, 2)),
    dict(block_table=ints(0, 1)),
    dict(cu_seqlens=ints(0, 10)),
    dict(total=-1),
    dict(dtype=torch.float32),
    dict(dtype=None),  # int8 is no type to read back in
    dict(key_cache=cache(torch.float16), value_cache=cache(torch.float16)),
    dict(out=(torch.zeros(9, 2, 64, dtype=BF16), torch.zeros(9, 2, 64, dtype=BF16))),
    dict(out=(torch.zeros(10, 2, 64), torch.zeros(10, 2, 64)), dtype=None),
    dict(out=(torch.zeros(10, 2, 64, dtype=BF16), torch.zeros(10, 2, 64, dtype=torch.float16))),
    dict(out=(torch.zeros(10, 2, 64, dtype=torch.float16),) * 2),
    dict(out=(torch.zeros(10, 2, 64, dtype=BF16),) * 2),
    dict(out=(torch.zeros(10, 2, 64, dtype=BF16),
              torch.zeros(2, 10, 64, dtype=BF16).transpose(0, 1))),
], ids=lambda c: "-".join(c))
def test_gather(no_launch, change):
    with pytest.raises((ValueError, UnsupportedConfig)):
        mx.gather_cache(**gather_args(**change))


# ---------------------------------------------------------------------------
# The C entries: argument lists of a good call, one entry changed

F16C, BF16C, E4M3C, INT8C = 0, 1, 2, 3
EUNSUPPORTED, EINVAL, EWORKSPACE = (native.MXFA_EUNSUPPORTED, native.MXFA_EINVAL,
                                    native.MXFA_EWORKSPACE)
no_gpu = pytest.mark.skipif(torch.cuda.is_available(),
                            reason="the addresses are made up: nothing may launch")


def at(n):
    return 1 << 20 | n << 12


def call_c(name, good, **change):
    assert set(change) <= set(good), set(change) - set(good)
    return getattr(native.library(), name)(*(good | change).values())


def prefill_c():
    return dict(
        q=at(1), q_st=8 * 64, q_sh=64, rows=10, cu=at(2), k=at(3), v=at(4), sp=16 * 128, st=128,
        sh=64, ks=0, ks_sp=0, ks_sh=0, vs=0, vs_sp=0, vs_sh=0, k1=0, v1=0, bt=at(5), bt_st=64,
        lens=at(6), out=at(7), o_st=8 * 64, o_sh=64, ws=at(8), ws_bytes=1 << 40, scale=0.1,
        causal=1, window=-1, cap=0.0, sinks=0, alibi=0, batch=2, hq=8, hkv=2, hd=64, ps=16,
        width=64, pages=8, dtype=BF16C, cdtype=BF16C, cus=256, stream=0)


@no_gpu
@pytest.mark.parametrize("change,rc", [
    (dict(rows=-1), EINVAL), (dict(batch=0), EINVAL), (dict(width=0), EINVAL),
    (dict(pages=0), EINVAL), (dict(cus=0), EINVAL), (dict(hkv=0), EINVAL),
    (dict(hd=96), EUNSUPPORTED), (dict(hq=7), EUNSUPPORTED), (dict(hq=34), EUNSUPPORTED),
    (dict(ps=24), EUNSUPPORTED), (dict(ps=8192), EUNSUPPORTED), (dict(dtype=2), EUNSUPPORTED),
    (dict(cdtype=F16C), EUNSUPPORTED), (dict(batch=16001), EUNSUPPORTED),
    (dict(width=1 << 27), EUNSUPPORTED), (dict(rows=1 << 30), EUNSUPPORTED),
    *[({x: 0}, EINVAL) for x in ("q", "cu", "k", "v", "bt", "lens", "out")],
    *[({x: at(9) + 2}, EINVAL) for x in ("q", "cu", "k", "v", "bt", "lens", "out", "ks", "vs",
                                         "k1", "v1", "sinks", "alibi")],
    (dict(q_st=8 * 64 + 4), EINVAL), (dict(q_sh=-64), EINVAL), (dict(sp=-2048), EINVAL),
    (dict(sh=60), EINVAL), (dict(bt_st=-1), EINVAL), (dict(o_st=0), EINVAL),
    (dict(o_sh=32), EINVAL), (dict(o_st=7 * 64), EINVAL), (dict(o_sh=66), EINVAL),
    (dict(window=-2), EINVAL), (dict(cap=-1.0), EINVAL), (dict(cap=float("inf")), EINVAL),
    (dict(cap=float("nan")), EINVAL), (dict(ws=0), EWORKSPACE), (dict(ws=at(8) + 4), EWORKSPACE),
    (dict(ws_bytes=1 << 20), EWORKSPACE),
], ids=str)
def test_prefill_entry(change, rc):
    assert call_c("mxfa_package_prefill_launch", prefill_c(), **change) == rc


def write_c():
    return dict(k=at(1), v=at(2), st=128, sh=64, kc=at(3), vc=at(4), sp=2048, ct=128, ch=64,
                ks=at(5), ks_sp=32, ks_sh=16, vs=at(6), vs_sp=32, vs_sh=16, slots=at(7), n=5,
                hkv=2, hd=64, ps=16, pages=8, dtype=BF16C, cdtype=INT8C, stream=0)


@no_gpu
@pytest.mark.parametrize("change,rc", [
    (dict(n=-1), EINVAL), (dict(hkv=0), EINVAL), (dict(pages=0), EINVAL), (dict(ps=0), EINVAL),
    (dict(ps=24), EUNSUPPORTED), (dict(hd=24), EUNSUPPORTED), (dict(hd=528), EUNSUPPORTED),
    (dict(dtype=E4M3C), EUNSUPPORTED), (dict(cdtype=BF16C), EUNSUPPORTED),
    *[({x: 0}, EINVAL) for x in ("k", "v", "kc", "vc", "ks", "vs", "slots")],
    *[({x: at(9) + 2}, EINVAL) for x in ("k", "v", "kc", "vc", "ks", "vs", "slots")],
    (dict(st=132), EINVAL), (dict(sh=-64), EINVAL), (dict(ct=136), EINVAL),
    (dict(sp=-2048), EINVAL), (dict(ks_sp=-1), EINVAL), (dict(vs_sh=-1), EINVAL),
    (dict(vc=at(3)), EINVAL), (dict(vs=at(5)), EINVAL),
], ids=str)
def test_write_entry(change, rc):
    assert call_c("mxfa_package_quantize_and_cache_launch", write_c(), **change) == rc


def gather_c():
    return dict(kc=at(1), vc=at(2), sp=2048, st=128, sh=64, ks=at(3), ks_sp=32, ks_sh=16,
                vs=at(4), vs_sp=32, vs_sh=16, k1=0, v1=0, bt=at(5), bt_st=3, cu=at(6), ko=at(7),
                vo=at(8), o_st=128, o_sh=64, batch=2, width=3, total=10, hkv=2, hd=64, ps=16,
                pages=8, dtype=BF16C, cdtype=INT8C, stream=0)


@no_gpu
@pytest.mark.parametrize("change,rc", [
    (dict(batch=0), EINVAL), (dict(width=0), EINVAL), (dict(total=-1), EINVAL),
    (dict(hkv=0), EINVAL), (dict(pages=0), EINVAL), (dict(ps=24), EUNSUPPORTED),
    (dict(hd=24), EUNSUPPORTED), (dict(dtype=INT8C), EUNSUPPORTED),
    (dict(cdtype=F16C), EUNSUPPORTED),
    *[({x: 0}, EINVAL) for x in ("kc", "vc", "bt", "cu", "ko", "vo")],
    *[({x: at(9) + 2}, EINVAL) for x in ("kc", "vc", "bt", "cu", "ko", "vo", "ks", "vs", "k1",
                                         "v1")],
    (dict(st=136), EINVAL), (dict(sh=-64), EINVAL), (dict(bt_st=-1), EINVAL),
    (dict(o_st=124), EINVAL), (dict(o_st=64), EINVAL), (dict(o_sh=56), EINVAL),
    (dict(vo=at(7)), EINVAL),
], ids=str)
def test_gather_entry(change, rc):
    assert call_c("mxfa_package_gather_cache_launch", gather_c(), **change) == rc


def decode_c():
    return dict(q=at(1), q_sb=8 * 64, q_st=0, q_sh=64, ql=1, causal=0, window=-1, sinks=0,
                cap=0.0, alibi=0, kc=at(2), vc=at(3), sp=2048, st=128, sh=64, ks=at(4), ks_sp=32,
                ks_sh=16, vs=at(5), vs_sp=32, vs_sh=16, bt=at(6), bt_st=64, lens=at(7), add=0,
                out=at(8), o_sb=8 * 64, o_st=0, o_sh=64, ws=at(9), ws_bytes=1 << 40, scale=0.1,
                batch=2, hq=8, hkv=2, hd=64, ps=16, width=64, pages=8, dtype=BF16C,
                kdtype=INT8C, ns=8, stream=0)


@no_gpu
@pytest.mark.parametrize("change,rc", [
    (dict(kdtype=BF16C), EUNSUPPORTED), (dict(dtype=INT8C), EUNSUPPORTED),
    (dict(hd=96), EUNSUPPORTED), (dict(hq=34), EUNSUPPORTED), (dict(ps=24), EUNSUPPORTED),
    (dict(batch=16001), EUNSUPPORTED), (dict(batch=0), EINVAL), (dict(ql=0), EINVAL),
    *[({x: 0}, EINVAL) for x in ("q", "kc", "vc", "bt", "lens", "out", "ks", "vs")],
    *[({x: at(10) + 2}, EINVAL) for x in ("q", "kc", "vc", "out", "ks", "vs")],
    (dict(ks_sp=-1), EINVAL), (dict(vs_sh=-1), EINVAL),
    (dict(window=-2), EINVAL), (dict(cap=-1.0), EINVAL), (dict(ws=0), EWORKSPACE),
    (dict(ws_bytes=16), EWORKSPACE),
], ids=str)
def test_decode_entry(change, rc):
    assert call_c("mxfa_package_decode_rows_launch", decode_c(), **change) == rc


@no_gpu
def test_empty_calls_launch_nothing():
    assert call_c("mxfa_package_prefill_launch", prefill_c(), rows=0, q=0) == native.MXFA_OK
    assert call_c("mxfa_package_quantize_and_cache_launch", write_c(), n=0) == native.MXFA_OK
    assert call_c("mxfa_package_gather_cache_launch", gather_c(), total=0) == native.MXFA_OK


def test_prefill_workspace():
    def size(batch, rows, hq, hkv, hd, ps, width, cus=256):
        out = ctypes.c_size_t()
        rc = native.library().mxfa_package_prefill_workspace_size(batch, rows, hq, hkv, hd, ps,
                                                                  width, cus, ctypes.byref(out))
        assert rc == native.MXFA_OK
        return out.value

    assert size(1, 1, 8, 2, 64, 16, 16) == 0  # 256 keys: no tile is cut
    # One long chunk fills the chip by itself.
    assert size(1, 100000, 32, 8, 128, 16, 8192) == 0
    # 2 * 64 pieces a kv head of 128 rows: outputs, sums, descriptors, the count.
    assert size(1, 1, 32, 8, 128, 16, 512) == 2 * 64 * 8 * (128 * (128 + 1) * 4 + 16) + 16
    # Nothing but the sizes of heads and the chip counts, so a captured call holds its share.
    assert size(300, 7000, 32, 8, 128, 16, 512) == size(1, 1, 32, 8, 128, 16, 99)
    assert native.library().mxfa_package_prefill_workspace_size(
        0, 1, 8, 2, 64, 16, 16, 256, ctypes.byref(ctypes.c_size_t())) == EINVAL


def test_pieces_fit_their_slots():
    """Row tiles cut into ceil(cost / most) pieces, most >= W / target: at most 2 * target of
    tiles that are cut, and at most `target` more than there are tiles."""
    g = torch.Generator().manual_seed(3)
    for _ in range(300):
        target = int(torch.randint(8, 513, (1,), generator=g))
        batch = int(torch.randint(1, 300, (1,), generator=g))
        tiles = torch.randint(0, 9, (batch,), generator=g, dtype=torch.int64)
        cost = (2.0 ** (torch.rand(batch, generator=g) * 17)).long()
        work = (tiles * cost).float().sum().item()
        most = max(256, int(min(work * 1.001 / target + 1, 2e9)))
        pieces = torch.where(cost > most, (cost + most - 1) // most, torch.ones_like(cost))
        cut = tiles * torch.where(pieces > 1, pieces, torch.zeros_like(pieces))
        assert int(cut.sum()) <= 2 * target
        assert int((tiles * (pieces - 1)).sum()) <= target
