"""Attention over a paged cache and the 8-bit cache, in 64 bits on the CPU, with bounds on
what 16-bit weights and outputs may be off by."""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def half_step(dtype: torch.dtype) -> float:
    """Largest relative error of one rounding to nearest."""
    return torch.finfo(dtype).eps / 2


@dataclass
class Paged:
    """B sequences' keys in shuffled pages; ks, vs: scales [pages, HKV, PS] or None."""

    kc: torch.Tensor
    vc: torch.Tensor
    ks: torch.Tensor | None
    vs: torch.Tensor | None
    table: torch.Tensor
    lens: torch.Tensor

    def to(self, device):
        move = lambda t: None if t is None else t.to(device)  # noqa: E731
        return Paged(*(move(t) for t in (self.kc, self.vc, self.ks, self.vs, self.table,
                                         self.lens)))


def quantise(x: torch.Tensor, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of rows x [..., HD], 32-bit arithmetic on the CPU."""
    x = x.float()
    top = torch.full((), TOP[dtype])
    scale = (x.abs().amax(-1) / top).clamp(min=2.0 ** -126)
    scale = torch.where(scale.isfinite(), scale, torch.full_like(scale, math.nan))
    y = (x / scale[..., None]).clamp(-TOP[dtype], TOP[dtype]).nan_to_num(0.0)
    return (y.round() if dtype == torch.int8 else y).to(dtype), scale


def make_paged(lens, hkv, hd, dtype, ps, *, codes=None, seed=0, width=None, fill=float("nan")):
    """Random keys; everything that no sequence holds is ``fill`` (codes: their largest)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // ps) for n in lens]
    pages = sum(need) + 3
    perm = torch.randperm(pages, generator=g)
    width = width or max(1, max(need))
    table = torch.randint(0, pages, (len(lens), width), generator=g, dtype=torch.int32)
    live = torch.zeros(pages, ps, dtype=torch.bool)
    at = 0
    for b, n in enumerate(need):
        own = perm[at:at + n]
        table[b, :n] = own.to(torch.int32)
        at += n
        flat = torch.arange(n * ps) < lens[b]
        live[own] = flat.view(n, ps)
    sides = []
    for _ in range(2):
        x = torch.randn(pages, ps, hkv, hd, generator=g).to(dtype)
        if codes is None:
            x[~live] = fill
            sides.append((x, None))
            continue
        c, s = quantise(x * torch.exp(torch.randn(pages, ps, hkv, 1, generator=g)).to(dtype), codes)
        c.view(torch.uint8)[~live] = 0x7F  # e4m3fn: NaN
        s[~live] = fill
        sides.append((c, s.permute(0, 2, 1).contiguous()))
    (kc, ks), (vc, vs) = sides
    return Paged(kc, vc, ks, vs, table, torch.tensor(lens, dtype=torch.int32))


def rows_of(p: Paged, b: int, k_scale=1.0, v_scale=1.0):
    """K and V rows [L, HKV, HD] of sequence b in float64."""
    n, ps = int(p.lens[b]), p.kc.shape[1]
    pos = torch.arange(n)
    page, off = p.table[b].long()[pos // ps], pos % ps
    k, v = p.kc.double()[page, off] * k_scale, p.vc.double()[page, off] * v_scale
    if p.ks is not None:
        k = k * p.ks[page, :, off].double()[..., None]
        v = v * p.vs[page, :, off].double()[..., None]
    return k, v


def attend(q, k, v, scale, *, causal=True, window=-1, softcap=0.0, sinks=None, alibi=None,
           weight_step=0.0, out_step=0.0):
    """(out, bound) [N, HQ, HD] in float64 of q [N, HQ, HD] at the last N of the keys' L
    positions (before them where N > L).

    The bound: every weight rounded once (weight_step), the output once (out_step), scores
    of HD products summed in 32 bits (each at most HD + 4 roundings of 2^-24 of the sum of
    magnitudes, an exponent's error being the weight's relative error), and the sums over L
    keys in 32 bits; results below fp16's normal range to its step."""
    n, hq, hd = q.shape
    length, hkv = k.shape[0], k.shape[1]
    q = q.double()
    k = k.repeat_interleave(hq // hkv, dim=1)
    v = v.repeat_interleave(hq // hkv, dim=1)
    if length == 0:
        return torch.zeros(n, hq, hd, dtype=torch.float64), torch.zeros(n, hq, hd).double()
    kt = k.permute(1, 2, 0)
    x = q.transpose(0, 1) @ kt * scale  # [HQ, N, L]
    mag = (q.abs().transpose(0, 1) @ kt.abs() * abs(scale)).nan_to_num(0.0)
    if softcap > 0:
        x = softcap * torch.tanh(x / softcap)
    behind = (length - n + torch.arange(n))[:, None] - torch.arange(length)[None, :]
    if alibi is not None:
        far = alibi.double()[:, None, None] * behind.abs()
        x = x - far
        mag = mag + far
    hidden = torch.zeros(n, length, dtype=torch.bool)
    if causal:
        hidden |= behind < 0
    if window >= 0:
        hidden |= behind > window
    x = x.masked_fill(hidden, -math.inf)
    top = x.amax(-1, keepdim=True).nan_to_num(0.0, neginf=0.0)
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    none = hidden.all(-1)
    if sinks is not None:
        total = total + torch.exp(sinks.double()[:, None, None] - top)
    w = torch.where(none[None, :, None], 0.0, w / total.clamp(min=1e-300))
    seen = (~hidden)[None].expand_as(w)
    # A key that a row does not see contributes nothing, whatever it holds.
    vt = v.transpose(0, 1)
    if bool(torch.isfinite(vt).all()):
        out, size = w @ vt, w @ vt.abs()
    else:
        out = torch.where(seen[..., None], w[..., None] * vt[:, None], 0.0).sum(2)
        size = out.abs()
    off = mag.masked_fill(hidden, 0.0).amax(-1, keepdim=True) * (hd + 4) * 2.0 ** -24 * 2
    bound = size * (weight_step + off + (length + 8) * 2.0 ** -24) * (1 + out_step)
    bound = bound + out.abs() * out_step + 2.0 ** -24
    return out.transpose(0, 1), bound.transpose(0, 1)


def check(got, want, bound, what=""):
    """got within bound of want everywhere, NaN where want is."""
    got = got.double().cpu()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan), f"{what}: NaN in other places"
    err = (got - want).abs()[~nan]
    lim = bound[~nan]
    if err.numel():
        worst = (err / lim.clamp(min=1e-300)).max().item()
        assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"
