"""paged_prefill on the GPU against attention in 64 bits, within bounds that count its
roundings (paged_reference.attend)."""

from __future__ import annotations

import pytest
import torch

import mxflashattn_amd as mx
from mxflashattn_amd import native

from paged_reference import Paged, attend, check, half_step, make_paged, rows_of

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def weight_step(dtype, codes):
    # An fp16 call on 8-bit rows holds its weights in two bf16 (16 bits).
    return 2.0 ** -16 if dtype == F16 and codes is not None else half_step(dtype)


def packed_q(new, hq, hd, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(new), hq, hd, generator=g).to(dtype)
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
    return q, cu


def expected(q, new, p: Paged, scale, dtype, codes, k_scale=1.0, v_scale=1.0, **options):
    out, bound = [], []
    for b, part in enumerate(q.split(new)):
        k, v = rows_of(p, b, k_scale, v_scale)
        o, e = attend(part, k, v, scale, weight_step=weight_step(dtype, codes),
                      out_step=half_step(dtype), **options)
        out.append(o)
        bound.append(e)
    return torch.cat(out), torch.cat(bound)


def call(q, cu, p: Paged, scale, device, *, causal=True, window=-1, softcap=0.0, sinks=None,
         alibi=None, **more):
    d = p.to(device)
    move = lambda t: None if t is None else t.to(device)  # noqa: E731
    if p.ks is not None:
        more = {"k_scale": d.ks, "v_scale": d.vs, **more}
    return mx.paged_prefill(q.to(device), d.kc, d.vc, cu.to(device), d.table, d.lens, scale,
                            causal=causal, window_left=window, softcap=softcap,
                            sinks=move(sinks), alibi_slopes=move(alibi), **more)


def run_case(device, new, lens, hq, hkv, hd, dtype, ps, codes=None, seed=0, **options):
    p = make_paged(lens, hkv, hd, dtype, ps, codes=codes, seed=seed)
    q, cu = packed_q(new, hq, hd, dtype, seed + 1)
    scale = hd ** -0.5
    want, bound = expected(q, new, p, scale, dtype, codes, **options)
    got = call(q, cu, p, scale, device, **options)
    torch.cuda.synchronize()
    check(got, want, bound, f"new {new} lens {lens}")


SHAPES = [  # new tokens, keys
    ([1], [1]),
    ([2, 1, 5], [2, 9, 64]),
    ([17], [100]),
    ([0, 3, 0, 70], [5, 3, 0, 131]),
    ([64, 65, 63], [64, 65, 127]),
    ([300], [300]),
    ([129, 1, 33], [700, 513, 33]),
]


@pytest.mark.parametrize("new,lens", SHAPES, ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_lengths(device, new, lens, hd, dtype):
    run_case(device, new, lens, 8, 2, hd, dtype, 16)


@pytest.mark.parametrize("codes", [E4M3, INT8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("new,lens", SHAPES, ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_lengths_8bit(device, codes, new, lens, hd, dtype):
    run_case(device, new, lens, 8, 2, hd, dtype, 16, codes)


@pytest.mark.parametrize("gq", [1, 2, 3, 5, 7, 16])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_head_groups(device, gq, hd):
    run_case(device, [40, 1, 90], [77, 300, 90], 3 * gq, 3, hd, BF16, 32)


@pytest.mark.parametrize("ps", [1, 2, 8, 16, 64, 256])
@pytest.mark.parametrize("codes", [None, E4M3, INT8], ids=["wide", "e4m3", "int8"])
def test_page_sizes(device, ps, codes):
    run_case(device, [40, 7], [201, 130], 8, 4, 128, BF16, ps, codes)


OPTIONS = [
    {"causal": False},
    {"window": 0},
    {"window": 5},
    {"window": 100},
    {"window": 70, "causal": False},
    {"softcap": 3.0},
    {"sinks": True},
    {"alibi": True},
    {"window": 33, "softcap": 2.0, "sinks": True, "alibi": True},
]


@pytest.mark.parametrize("options", OPTIONS, ids=str)
@pytest.mark.parametrize("hd,codes", [(64, None), (128, None), (256, None), (128, INT8),
                                      (64, E4M3)])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_options(device, options, hd, codes, dtype):
    options = dict(options)
    g = torch.Generator().manual_seed(3)
    for name in ("sinks", "alibi"):
        if options.get(name):
            options[name] = torch.rand(8, generator=g) * (4.0 if name == "sinks" else 0.2)
    run_case(device, [130, 1, 20], [140, 400, 300], 8, 2, hd, dtype, 16, codes, **options)


@pytest.mark.parametrize("codes", [None, INT8], ids=["wide", "int8"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new,lens", [([1], [5000]), ([3, 1, 1, 40], [2000, 3001, 700, 900]),
                                      ([20], [4097])],
                         ids=lambda v: "-".join(map(str, v)))
def test_few_rows_many_keys(device, new, lens, hd, codes):
    """Row tiles cut into pieces of their keys, and joined."""
    run_case(device, new, lens, 8, 2, hd, BF16, 16, codes)


@pytest.mark.parametrize("options", [{"window": 1500}, {"sinks": True}, {"causal": False}], ids=str)
def test_pieces_with_options(device, options):
    options = dict(options)
    if options.get("sinks"):
        options["sinks"] = torch.linspace(-2, 5, 8)
    run_case(device, [30, 2], [3500, 2600], 8, 2, 128, F16, 16, **options)


def test_tokens_without_keys_are_zeros(device):
    """More new tokens than keys: those before the first key see none."""
    p = make_paged([3, 0], 2, 64, BF16, 16)
    q, cu = packed_q([7, 4], 4, 64, BF16)
    got = call(q, cu, p, 0.125, device)
    want, bound = expected(q, [7, 4], p, 0.125, BF16, None)
    check(got, want, bound)
    assert not got[:4].any() and not got[7:].any()


def test_rows_behind_the_last_sequence_stay(device):
    p = make_paged([40, 9], 2, 128, F16, 16).to(device)
    q, cu = packed_q([40, 2], 4, 128, F16)
    q = torch.cat([q, q[:6]]).to(device)
    out = torch.full_like(q, 7.0)
    got = mx.paged_prefill(q, p.kc, p.vc, cu.to(device), p.table, p.lens, 0.1, out=out)
    assert got is out and bool((out[42:] == 7.0).all()) and bool(out[:42].isfinite().all())


def test_rows_without_a_scale_reach_only_tokens_that_see_them(device):
    """A NaN key or value row (its scale NaN) makes later tokens NaN, no earlier one."""
    for codes in (E4M3, INT8):
        for side in ("ks", "vs"):
            p = make_paged([90], 2, 128, BF16, 16, codes=codes)
            scale = getattr(p, side)
            scale[p.table[0, 80 // 16], 1, 80 % 16] = float("nan")
            q, cu = packed_q([30], 4, 128, BF16)
            got = call(q, cu, p, 0.1, device).cpu()
            nan = got.isnan()
            assert bool(nan[20:, 2:].all()) and not bool(nan[:20].any())
            assert not bool(nan[:, :2].any())


@pytest.mark.parametrize("codes", [None, E4M3, INT8], ids=["16", "e4m3", "int8"])
@pytest.mark.parametrize("new,window", [(1, 40), (9, 3), (9, 0), (70, 40), (1, 700), (200, 150)])
def test_nan_ahead_of_the_window(device, codes, new, window):
    """Keys ahead of every token's window may hold anything: their pages may be another's."""
    length = 900
    p = make_paged([length], 2, 64, BF16, 16, codes=codes)
    q, cu = packed_q([new], 8, 64, BF16)
    want, bound = expected(q, [new], p, 0.125, BF16, codes, window=window)
    gone = torch.arange(length - new - window)
    page, off = p.table[0].long()[gone // 16], gone % 16
    for x, s in ((p.kc, p.ks), (p.vc, p.vs)):
        if codes is None:
            x[page, off] = float("nan")
        else:
            x.view(torch.uint8)[page, off] = 0x7F
            s[page, :, off] = float("nan")
    check(call(q, cu, p, 0.125, device, window=window), want, bound)


def test_windows_past_the_positions(device):
    """Windows of up to 2^31 - 1 and more hide nothing, with tokens ahead of the first key too."""
    p = make_paged([30, 100], 2, 64, BF16, 16)
    q, cu = packed_q([37, 20], 8, 64, BF16)
    want, bound = expected(q, [37, 20], p, 0.125, BF16, None)
    for window in (100, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1, 2 ** 32 + 3):
        check(call(q, cu, p, 0.125, device, window=window), want, bound, f"window {window}")


def test_scale_of_the_whole_cache(device):
    p = make_paged([150, 20], 2, 128, BF16, 16, fill=0.0)
    p = Paged(p.kc.to(E4M3), p.vc.to(E4M3), None, None, p.table, p.lens)
    q, cu = packed_q([33, 20], 8, 128, BF16)
    ks, vs = (torch.tensor([x], device=device) for x in (0.5, 3.0))
    want, bound = expected(q, [33, 20], p, 0.1, BF16, E4M3, 0.5, 3.0)
    check(call(q, cu, p, 0.1, device, k_scale=ks, v_scale=vs), want, bound)
    check(call(q, cu, p, 0.1, device, k_scale=0.5, v_scale=3.0), want, bound)


def test_strides(device):
    """q a slice of a fused projection, heads-first pages, a strided output, int64 metadata."""
    p = make_paged([130, 50], 4, 64, F16, 16)
    q, cu = packed_q([60, 50], 8, 64, F16)
    want, bound = expected(q, [60, 50], p, 0.125, F16, None)
    d = p.to(device)
    fused = torch.zeros(110, 16, 64, dtype=F16, device=device)
    fused[:, 4:12] = q.to(device)
    heads_first = [c.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for c in (d.kc, d.vc)]
    out = torch.zeros(110, 9, 64, dtype=F16, device=device)
    got = mx.paged_prefill(fused[:, 4:12], *heads_first, cu.to(device).long(), d.table.long(),
                           d.lens.long(), 0.125, out=out[:, 1:])
    check(got, want, bound)
    assert not out[:, 0].any()
    odd = torch.zeros(110 * 8 * 64 + 1, dtype=F16, device=device)[1:].view(110, 8, 64)
    check(mx.paged_prefill(q.to(device), d.kc, d.vc, cu.to(device), d.table, d.lens, 0.125,
                           out=odd), want, bound)


def test_agrees_with_the_decode_of_one_token(device):
    p = make_paged([1000, 33, 700], 4, 128, BF16, 16).to(device)
    q, cu = packed_q([1, 1, 1], 16, 128, BF16)
    a = mx.paged_prefill(q.to(device), p.kc, p.vc, cu.to(device), p.table, p.lens, 0.1)
    b = mx.paged_decode_split(q.to(device), p.kc, p.vc, p.table, p.lens, 0.1)
    # Both round the weights and the output once.
    assert float((a.double() - b.double()).norm() / b.double().norm()) < 4 * half_step(BF16)


def test_captured_with_other_lengths(device):
    """A captured call replays with the lengths, offsets and pages of the moment."""
    hq, hkv, hd = 8, 2, 128
    p = make_paged([2000, 900], hkv, hd, BF16, 16, fill=0.0)
    d = p.to(device)
    q, cu = packed_q([30, 60], hq, hd, BF16)
    qd, cud = q.to(device), cu.to(device)
    out = torch.zeros_like(qd)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        mx.paged_prefill(qd, d.kc, d.vc, cud, d.table, d.lens, 0.1, out=out)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        mx.paged_prefill(qd, d.kc, d.vc, cud, d.table, d.lens, 0.1, out=out)
    for new, lens in (([30, 60], [2000, 900]), ([80, 10], [90, 10]), ([1, 89], [1800, 89]),
                      ([0, 90], [0, 700])):
        cud.copy_(torch.tensor([0, new[0], 90], dtype=torch.int32))
        d.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        now = Paged(p.kc, p.vc, None, None, p.table, torch.tensor(lens, dtype=torch.int32))
        want, bound = expected(q, new, now, 0.1, BF16, None)
        check(out, want, bound, f"replay {new} {lens}")


def test_streams_do_not_share_a_workspace(device):
    cases = []
    for seed in range(3):
        p = make_paged([3000, 40], 2, 64, F16, 16, seed=seed)
        q, cu = packed_q([2, 40], 4, 64, F16, seed)
        cases.append((p, q, cu, expected(q, [2, 40], p, 0.125, F16, None)))
    streams = [torch.cuda.Stream() for _ in cases]
    moved = [(p.to(device), q.to(device), cu.to(device)) for p, q, cu, _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for s, (p, q, cu) in zip(streams, moved):
            with torch.cuda.stream(s):
                outs.append(mx.paged_prefill(q, p.kc, p.vc, cu, p.table, p.lens, 0.125))
        torch.cuda.synchronize()
        for out, (*_, (want, bound)) in zip(outs, cases):
            check(out, want, bound)


@pytest.mark.parametrize("torch_op", [True, False], ids=["op", "ctypes"])
def test_threads_on_one_stream(device, monkeypatch, torch_op):
    """Calls of several threads on one stream: each pair of launches stays together."""
    from concurrent.futures import ThreadPoolExecutor

    monkeypatch.setattr(native, "USE_TORCH_OP", torch_op)
    stream = torch.cuda.Stream()
    calls = []
    for seed in range(4):
        codes = INT8 if seed % 2 else None
        p = make_paged([6000, 3000], 2, 128, BF16, 16, codes=codes, seed=seed).to(device)
        q, cu = packed_q([8, 20], 8, 128, BF16, seed)
        calls.append((q.to(device), p, cu.to(device)))

    def run(i):
        q, p, cu = calls[i]
        if i == 3:  # the decode of the same rows
            return mx.paged_decode_split(q[:2], p.kc, p.vc, p.table, p.lens, 0.1, num_splits=64,
                                         k_scale=p.ks, v_scale=p.vs)
        return mx.paged_prefill(q, p.kc, p.vc, cu, p.table, p.lens, 0.1, k_scale=p.ks,
                                v_scale=p.vs)

    def many(i):
        with torch.cuda.stream(stream):
            return [run(i) for _ in range(25)]

    with torch.cuda.stream(stream):
        want = [run(i) for i in range(4)]
    torch.cuda.synchronize()
    with ThreadPoolExecutor(4) as pool:
        got = list(pool.map(many, range(4)))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


@pytest.mark.parametrize("torch_op", [True, False], ids=["op", "ctypes"])
def test_captured_calls_side_by_side(device, monkeypatch, torch_op):
    """Two graphs captured on one stream, replayed on two at once beside eager calls on the
    first: cut tiles' pieces of the one never meet the other's."""
    monkeypatch.setattr(native, "USE_TORCH_OP", torch_op)
    capture, other = torch.cuda.Stream(), torch.cuda.Stream()
    calls = []
    for seed in (3, 4):
        p = make_paged([6000, 3000], 2, 128, BF16, 16, seed=seed).to(device)
        q, cu = packed_q([8, 20], 8, 128, BF16, seed)
        calls.append((q.to(device), p, cu.to(device)))

    def run(i):
        q, p, cu = calls[i]
        return mx.paged_prefill(q, p.kc, p.vc, cu, p.table, p.lens, 0.1)

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


def test_pages_past_4_gib(device):
    """Byte offsets into the cache that 32 bits do not hold."""
    hkv, hd, ps = 2, 128, 16
    pages = (5 << 30) // (ps * hkv * hd * 2)
    kc = torch.empty(pages, ps, hkv, hd, dtype=BF16, device=device)
    vc = torch.empty_like(kc)
    small = make_paged([200], hkv, hd, BF16, ps, fill=0.0)
    table = small.table.clone()
    n = 13
    far = torch.linspace(pages // 2, pages - 1, n).long()
    kc[far.to(device)] = small.kc[small.table[0, :n].long()].to(device)
    vc[far.to(device)] = small.vc[small.table[0, :n].long()].to(device)
    table[0, :n] = far.to(torch.int32)
    q, cu = packed_q([50], 4, hd, BF16)
    want, bound = expected(q, [50], small, 0.1, BF16, None)
    got = mx.paged_prefill(q.to(device), kc, vc, cu.to(device), table.to(device),
                           small.lens.to(device), 0.1)
    check(got, want, bound)


def test_empty_call(device):
    p = make_paged([5], 2, 64, F16, 16).to(device)
    q = torch.zeros(0, 4, 64, dtype=F16, device=device)
    cu = torch.zeros(2, dtype=torch.int32, device=device)
    assert mx.paged_prefill(q, p.kc, p.vc, cu, p.table, p.lens, 0.1).shape == (0, 4, 64)


def test_many_sequences(device):
    """More sequences than threads of a workgroup."""
    new = [1 + (i * 7) % 3 for i in range(700)]
    lens = [n + (i * 13) % 40 for i, n in enumerate(new)]
    run_case(device, new, lens, 4, 2, 64, F16, 16)
