"""The 8-bit cache on the GPU: rows written (codes and scales equal to 32-bit arithmetic),
read back, and decoded against attention in 64 bits."""

from __future__ import annotations

import pytest
import torch

import mxflashattn_amd as mx
from mxflashattn_amd import native

from paged_reference import Paged, attend, check, half_step, make_paged, quantise, rows_of

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
KINDS = pytest.mark.parametrize("codes", [E4M3, INT8], ids=["e4m3", "int8"])
TYPES = pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])


def caches(pages, ps, hkv, hd, codes, device, mark=0x11):
    c = [torch.full((pages, ps, hkv, hd), mark, dtype=torch.uint8, device=device).view(codes)
         for _ in range(2)]
    s = [torch.full((pages, hkv, ps), 9.0, device=device) for _ in range(2)]
    return c, s


def bits(t):
    return t.cpu().contiguous().view(torch.uint8)


def check_written(got_codes, got_scales, rows, slots, ps, codes, mark=0x11):
    """The slots hold the rows' codes and scales, everything else what it held."""
    want_c, want_s = quantise(rows.cpu(), codes)
    full_c = torch.full_like(bits(got_codes), mark)
    full_s = torch.full_like(got_scales.cpu(), 9.0)
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < got_codes.shape[0] * ps:
            full_c[slot // ps, slot % ps] = want_c[t].view(torch.uint8)
            full_s[slot // ps, :, slot % ps] = want_s[t]
    assert torch.equal(got_scales.cpu().view(torch.int32), full_s.view(torch.int32)) or (
        torch.equal(got_scales.cpu().nan_to_num(-1.0), full_s.nan_to_num(-1.0)))
    assert torch.equal(bits(got_codes), full_c)


@KINDS
@TYPES
@pytest.mark.parametrize("n,hkv,hd,ps", [(1, 1, 64, 16), (3, 2, 128, 1), (77, 8, 128, 16),
                                         (130, 5, 256, 64), (9, 3, 16, 8), (31, 2, 48, 16),
                                         (5, 1, 512, 4096), (300, 7, 80, 32)])
def test_write(device, codes, dtype, n, hkv, hd, ps):
    g = torch.Generator().manual_seed(n)
    pages = -(-n // ps) + 2
    key, value = ((torch.randn(n, hkv, hd, generator=g)
                   * torch.exp(2 * torch.randn(n, hkv, 1, generator=g))).to(dtype)
                  for _ in range(2))
    slots = torch.randperm(pages * ps, generator=g)[:n]
    if n > 4:
        slots[2] = -1
        slots[4] = pages * ps + 3  # past the cache
    (kc, vc), (ks, vs) = caches(pages, ps, hkv, hd, codes, device)
    mx.quantize_and_cache(key.to(device), value.to(device), kc, vc, ks, vs, slots.to(device))
    torch.cuda.synchronize()
    check_written(kc, ks, key, slots, ps, codes)
    check_written(vc, vs, value, slots, ps, codes)


@KINDS
@TYPES
def test_write_of_special_rows(device, codes, dtype):
    """Zeros, subnormals, the largest values, halfway cases, infinities and NaN."""
    hd, big = 64, torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    x = torch.zeros(10, 1, hd)
    x[1, 0, 3] = tiny
    x[2, 0] = torch.linspace(-tiny, tiny, hd) / 7
    x[3, 0] = torch.linspace(-big, big, hd)
    x[4, 0] = torch.arange(hd) / 2 - 16.0   # halves
    x[4, 0, 0] = 127.0
    x[5, 0, 9] = float("inf")
    x[6, 0, 11] = float("nan")
    x[7, 0, 63] = float("-inf")
    x[8, 0] = torch.linspace(-1, 1, hd) * 448
    x[9, 0] = -0.0
    x = x.to(dtype)
    (kc, vc), (ks, vs) = caches(2, 16, 1, hd, codes, device)
    slots = torch.arange(10) + 3
    mx.quantize_and_cache(x.to(device), x.flip(0).contiguous().to(device), kc, vc, ks, vs,
                          slots.to(device))
    torch.cuda.synchronize()
    check_written(kc, ks, x, slots, 16, codes)
    check_written(vc, vs, x.flip(0), slots, 16, codes)
    # (linspace between the largest bf16 values passes through infinities.)
    assert torch.equal(ks[0, 0, 3:13].isnan().cpu(), ~x[:, 0].isfinite().all(-1))
    assert bool(ks[0, 0, 3 + 5:3 + 8].isnan().all())


@KINDS
def test_write_of_strided_rows(device, codes):
    """Slices of a fused projection, rows with other strides, scales of another layout."""
    n, hkv, hd, ps = 40, 4, 128, 16
    qkv = torch.randn(n, 3 * hkv, hd, generator=torch.Generator().manual_seed(0)).to(BF16)
    slots = torch.randperm(64, generator=torch.Generator().manual_seed(1))[:n]
    (kc, vc), _ = caches(4, ps, hkv, hd, codes, device)
    both = torch.full((2, hkv, 4, ps), 9.0, device=device)
    ks, vs = both[0].transpose(0, 1), both[1].transpose(0, 1)
    dev = qkv.to(device)
    mx.quantize_and_cache(dev[:, hkv:2 * hkv], dev[:, 2 * hkv:], kc, vc, ks, vs,
                          slots.to(device).to(torch.int32))
    check_written(kc, ks, qkv[:, hkv:2 * hkv], slots, ps, codes)
    check_written(vc, vs, qkv[:, 2 * hkv:], slots, ps, codes)
    (kc, vc), (ks, vs) = caches(4, ps, hkv, hd, codes, device)
    odd = qkv[:, :hkv].permute(1, 0, 2).contiguous().permute(1, 0, 2)
    flat = torch.zeros(odd.numel() + 1, dtype=BF16, device=device)[1:].view(n, hkv, hd)
    flat.copy_(odd)  # not 16-byte aligned
    mx.quantize_and_cache(flat, odd.to(device), kc, vc, ks, vs, slots.to(device))
    check_written(kc, ks, odd, slots, ps, codes)
    check_written(vc, vs, odd, slots, ps, codes)


def same(a, b):
    differ = int((a.cpu() != b).sum())
    assert differ == 0, f"{differ} of {b.numel()} values differ"


def read_rows(p: Paged, lens, dtype, k_scale=1.0, v_scale=1.0):
    """What reading back gives: code * scale in 32 bits, rounded once."""
    parts = []
    for codes, scale, one in ((p.kc, p.ks, k_scale), (p.vc, p.vs, v_scale)):
        rows = []
        for b, n in enumerate(lens):
            ps = codes.shape[1]
            pos = torch.arange(n)
            page, off = p.table[b].long()[pos // ps], pos % ps
            if codes.dtype == dtype:
                rows.append(codes[page, off])
                continue
            x = codes.float()[page, off]
            x = x * scale[page, :, off][..., None] if scale is not None else x * one
            rows.append(x.to(dtype))
        parts.append(torch.cat(rows))
    return parts


@pytest.mark.parametrize("codes", [None, E4M3, INT8], ids=["wide", "e4m3", "int8"])
@TYPES
@pytest.mark.parametrize("lens,hkv,hd,ps", [([1], 1, 64, 16), ([5, 0, 33, 16], 2, 128, 16),
                                            ([200, 1, 77], 8, 128, 8), ([300], 5, 256, 64),
                                            ([40, 41], 3, 48, 1), ([9] * 300, 1, 16, 4)])
def test_read_back(device, codes, dtype, lens, hkv, hd, ps):
    p = make_paged(lens, hkv, hd, dtype, ps, codes=codes, seed=5)
    want = read_rows(p, lens, dtype)
    d = p.to(device)
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32,
                      device=device)
    got = mx.gather_cache(d.kc, d.vc, d.table, cu, sum(lens), k_scale=d.ks, v_scale=d.vs,
                          dtype=dtype)
    for a, b in zip(got, want):
        same(a, b)
    # Into strided tensors with rows behind the last sequence, which stay.
    room = torch.full((2, sum(lens) + 3, hkv + 1, hd), 5.0, dtype=dtype, device=device)
    mx.gather_cache(d.kc, d.vc, d.table, cu, sum(lens) + 3, k_scale=d.ks, v_scale=d.vs,
                    out=(room[0, :, 1:], room[1, :, 1:]))
    for a, b in zip(room.cpu(), want):
        same(a[:sum(lens), 1:], b)
        assert bool((a[sum(lens):] == 5.0).all()) and bool((a[:, 0] == 5.0).all())


def test_read_back_of_a_scale_for_the_whole_cache(device):
    p = make_paged([70, 3], 2, 64, F16, 16, fill=0.0)
    p = Paged(p.kc.to(E4M3), p.vc.to(E4M3), None, None, p.table, p.lens)
    d = p.to(device)
    cu = torch.tensor([0, 70, 73], dtype=torch.int32, device=device)
    got = mx.gather_cache(d.kc, d.vc, d.table, cu, 73, k_scale=0.3,
                          v_scale=torch.tensor([0.7], device=device), dtype=BF16)
    want = read_rows(p, [70, 3], BF16, torch.tensor(0.3), torch.tensor(0.7))
    for a, b in zip(got, want):
        same(a, b)


def test_written_rows_read_back(device):
    """What is read back is what quantising stands for: within half a code's step."""
    n, hkv, hd, ps = 50, 4, 128, 16
    g = torch.Generator().manual_seed(2)
    x = torch.randn(n, hkv, hd, generator=g).to(BF16)
    for codes in (E4M3, INT8):
        (kc, vc), (ks, vs) = caches(4, ps, hkv, hd, codes, device)
        table = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device=device)
        pos = torch.arange(n)
        slots = (table.cpu()[0].long()[pos // ps] * ps + pos % ps).to(device)
        mx.quantize_and_cache(x.to(device), x.to(device), kc, vc, ks, vs, slots)
        cu = torch.tensor([0, n], dtype=torch.int32, device=device)
        k, v = mx.gather_cache(kc, vc, table, cu, n, k_scale=ks, v_scale=vs, dtype=F16)
        assert torch.equal(k, v)
        top = x.double().abs().amax(-1, keepdim=True)
        # int8: half a step of top / 127; e4m3fn: half a step relative, or of its least
        # normal (2^-6 of 448 times the scale); then fp16's rounding of the result.
        step = (top / 127 / 2 if codes == INT8
                else torch.maximum(x.double().abs() * 2.0 ** -4, top / 448 * 2.0 ** -10))
        lim = (step + x.double().abs() * half_step(F16)) * (1 + 1e-3) + 2.0 ** -25
        assert bool(((k.cpu().double() - x.double()).abs() <= lim).all())


# ---------------------------------------------------------------------------
# Decode


def run_decode(device, lens, hq, hkv, hd, dtype, ps, codes, ql=1, num_splits=None, seed=0,
               options=None, kernel=None):
    options = options or {}
    p = make_paged(lens, hkv, hd, dtype, ps, codes=codes, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lens), ql, hq, hd, generator=g).to(dtype)
    step = 2.0 ** -16 if dtype == F16 else half_step(dtype)
    parts = [attend(q[b], *rows_of(p, b), hd ** -0.5, weight_step=step,
                    out_step=half_step(dtype), **options) for b in range(len(lens))]
    want, bound = (torch.stack(t) for t in zip(*parts))
    d = p.to(device)
    move = lambda t: None if t is None else t.to(device)  # noqa: E731
    got = mx.paged_decode_split(
        q.to(device), d.kc, d.vc, d.table, d.lens, hd ** -0.5, k_scale=d.ks, v_scale=d.vs,
        num_splits=num_splits, causal=options.get("causal", True),
        window_left=options.get("window", -1), softcap=options.get("softcap", 0.0),
        sinks=move(options.get("sinks")), alibi_slopes=move(options.get("alibi")))
    torch.cuda.synchronize()
    check(got, want, bound, f"lens {lens} ql {ql}")


@KINDS
@TYPES
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens", [[1], [16, 17, 0, 15], [700, 33], [2500, 3, 900]],
                         ids=lambda v: "-".join(map(str, v)))
def test_decode(device, codes, dtype, hd, lens):
    run_decode(device, lens, 8, 2, hd, dtype, 16, codes)


@KINDS
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("gq,hkv", [(1, 8), (3, 5), (7, 1), (16, 2), (4, 8)])
def test_decode_head_groups(device, codes, hd, gq, hkv):
    run_decode(device, [300, 1100], gq * hkv, hkv, hd, BF16, 32, codes)


@KINDS
@pytest.mark.parametrize("ps", [1, 4, 8, 16, 64, 256])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_decode_page_sizes(device, codes, ps, hd):
    run_decode(device, [99, 500, 1], 8, 2, hd, BF16, ps, codes)


@KINDS
@TYPES
@pytest.mark.parametrize("options", [{"window": 0}, {"window": 77}, {"softcap": 2.0},
                                     {"sinks": True}, {"alibi": True},
                                     {"window": 300, "softcap": 4.0, "sinks": True,
                                      "alibi": True}], ids=str)
@pytest.mark.parametrize("ql", [1, 3])
def test_decode_options(device, codes, dtype, options, ql):
    options = dict(options)
    for name in ("sinks", "alibi"):
        if options.get(name):
            options[name] = torch.linspace(0.0, 3.0 if name == "sinks" else 0.1, 8)
    for hd in (64, 128, 256):
        run_decode(device, [400, 1000], 8, 2, hd, dtype, 16, codes, ql=ql, options=options)


@KINDS
@pytest.mark.parametrize("ql,causal", [(2, True), (4, False), (9, True)])
def test_decode_tokens(device, codes, ql, causal):
    """Several tokens of a sequence, also more than one launch takes."""
    run_decode(device, [300, 900, 70], 8, 2, 128, BF16, 16, codes, ql=ql,
               options={"causal": causal})


@KINDS
@pytest.mark.parametrize("num_splits", [1, 7, 64, native.SPLITS_PER_SEQUENCE])
def test_decode_splits(device, codes, num_splits):
    run_decode(device, [300, 900, 0, 17], 16, 4, 128, BF16, 16, codes, num_splits=num_splits)


@KINDS
def test_decode_of_many_sequences(device, codes):
    lens = [(i * 37) % 90 for i in range(300)]
    run_decode(device, lens, 4, 1, 64, F16, 16, codes, num_splits=200)


@KINDS
def test_decode_of_rows_without_a_scale(device, codes):
    """NaN for the tokens and heads that see the row only."""
    for side in ("ks", "vs"):
        p = make_paged([60, 60], 2, 128, BF16, 16, codes=codes)
        getattr(p, side)[p.table[0, 3], 1, 10] = float("nan")  # position 58 of sequence 0
        q = torch.randn(2, 3, 4, 128, generator=torch.Generator().manual_seed(0)).to(BF16)
        d = p.to(device)
        got = mx.paged_decode_split(q.to(device), d.kc, d.vc, d.table, d.lens, 0.1, k_scale=d.ks,
                                    v_scale=d.vs, causal=True).cpu()
        nan = got.isnan()
        assert bool(nan[0, 1:, 2:].all())
        assert not bool(nan[0, 0].any()) and not bool(nan[0, :, :2].any())
        assert not bool(nan[1].any())


@pytest.mark.parametrize("torch_op", [True, False], ids=["op", "ctypes"])
def test_captured_decodes_side_by_side(device, monkeypatch, torch_op):
    """Two graphs captured on one stream, replayed on two at once beside eager calls."""
    monkeypatch.setattr(native, "USE_TORCH_OP", torch_op)
    capture, other = torch.cuda.Stream(), torch.cuda.Stream()
    calls = []
    for seed in (3, 4):
        p = make_paged([6000, 3000, 5000], 2, 128, BF16, 16, codes=INT8, seed=seed).to(device)
        q = torch.randn(3, 8, 128, generator=torch.Generator().manual_seed(seed)).to(BF16)
        calls.append((q.to(device), p))

    def run(i):
        q, p = calls[i]
        return mx.paged_decode_split(q, p.kc, p.vc, p.table, p.lens, 0.1, num_splits=64,
                                     k_scale=p.ks, v_scale=p.vs)

    with torch.cuda.stream(capture):
        want = [run(0).clone(), run(1).clone()]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=capture):
            outs.append(run(i))
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graphs[1].replay()
        with torch.cuda.stream(capture):
            graphs[0].replay()
            eager = run(1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        assert torch.equal(eager, want[1])


# ---------------------------------------------------------------------------
# The run of them


@KINDS
def test_prompt_then_tokens(device, codes):
    """A prompt in two chunks, then three tokens, through the write, the chunk attention,
    the decode and the read-back of one cache."""
    hq, hkv, hd, ps, dtype = 8, 2, 128, 16, BF16
    g = torch.Generator().manual_seed(8)
    n = 150
    q, k, v = (torch.randn(n, h, hd, generator=g).to(dtype) for h in (hq, hkv, hkv))
    (kc, vc), (ks, vs) = caches(12, ps, hkv, hd, codes, device)
    table = torch.randperm(12, generator=g)[:10].to(torch.int32)[None]
    pos = torch.arange(n)
    slots = (table[0].long()[pos // ps] * ps + pos % ps).to(device)
    outs = []
    qd, kd, vd, td = (t.to(device) for t in (q, k, v, table))
    for a, b in ((0, 100), (100, 147), (147, 148), (148, 149), (149, 150)):
        mx.quantize_and_cache(kd[a:b], vd[a:b], kc, vc, ks, vs, slots[a:b])
        lens = torch.tensor([b], dtype=torch.int32, device=device)
        if b - a > 1:
            cu = torch.tensor([0, b - a], dtype=torch.int32, device=device)
            outs.append(mx.paged_prefill(qd[a:b], kc, vc, cu, td, lens, 0.1, k_scale=ks,
                                         v_scale=vs))
        else:
            outs.append(mx.paged_decode_split(qd[a:b], kc, vc, td, lens, 0.1, k_scale=ks,
                                              v_scale=vs))
    ck, sk = quantise(k, codes)
    cv, sv = quantise(v, codes)
    want, bound = attend(q, ck.double() * sk.double()[..., None],
                         cv.double() * sv.double()[..., None], 0.1,
                         weight_step=half_step(dtype), out_step=half_step(dtype))
    check(torch.cat(outs), want, bound)
    cu = torch.tensor([0, n], dtype=torch.int32, device=device)
    back, _ = mx.gather_cache(kc, vc, td, cu, n, k_scale=ks, v_scale=vs, dtype=dtype)
    assert torch.equal(back.cpu(), (ck.float() * sk[..., None]).to(dtype))
