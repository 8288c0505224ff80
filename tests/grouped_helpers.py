"""64-bit references and error bounds of the products whose weight is picked by the row."""
from __future__ import annotations

import math

import torch

DTYPES = [torch.float16, torch.bfloat16]


def counts_to_offsets(counts, dtype=torch.int32, first=0):
    """Row numbers [E + 1] on the GPU of groups with these counts, the first at row `first`."""
    return (torch.tensor([0] + list(counts), device="cuda").cumsum(0) + first).to(dtype)


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def stacked(E, K, N, dtype, seed, stored="kn"):
    """A logical [E, K, N] weight, row-major or as the transposed view of [E, N, K] storage."""
    if stored == "kn":
        return randn((E, K, N), dtype, seed, K ** -0.5 if K else 1.0)
    return randn((E, N, K), dtype, seed, K ** -0.5 if K else 1.0).transpose(1, 2)


def act64(v, act):
    if act == "relu":
        return v.clamp_min(0.0)
    if act == "gelu":
        return v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
    return v


def half_step(dtype):
    """The relative error of one rounding to nearest."""
    return torch.finfo(dtype).eps / 2


def sum_error(steps, magnitude):
    """Error of an fp32 sum of exact 16-bit products on the tensor cores.

    16 products join the accumulator per instruction, and every addition errs
    by at most one unit in the last place (2^-23, a truncation) of a partial
    sum, which the sum of the magnitudes bounds: steps / 16 instructions, plus
    16 additions inside one, plus 8 for joining the pieces of a split sum.
    """
    return (math.ceil(steps / 16) + 24) * 2.0 ** -23 * magnitude


def act_error(v, err, act):
    """The error of act(v) when v errs by `err`: |gelu'| <= 1.13, and erff and
    the products around it err by a few units of |v|."""
    if act == "gelu":
        return 1.13 * err + 8 * 2.0 ** -24 * v.abs()
    return err


def rounded(ref, err, dtype):
    """Bound of |out - ref| once a value that errs by `err` is rounded to dtype."""
    tiny = torch.finfo(dtype).smallest_normal * half_step(dtype)   # half a step among the subnormals
    return err + half_step(dtype) * (ref.abs() + err) + tiny


def check(out, ref, tol, what=""):
    got = out.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    off = (got - ref).abs()
    ok = off <= tol
    assert bool(ok.all()), (f"{what}: {int((~ok).sum())} of {ok.numel()} values off, worst "
                            f"{float((off / tol).nan_to_num(posinf=1e9, nan=1e9).max()):.3g} times the bound")


def ref_grouped(A, B, offsets, bias=None, act="none"):
    """(reference, bound) of grouped_gemm into a new output."""
    T, N = A.shape[0], B.shape[2]
    ref = torch.zeros((T, N), dtype=torch.float64, device=A.device)
    tol = torch.zeros_like(ref)
    off = offsets.tolist()
    for e in range(B.shape[0]):
        s = slice(off[e], off[e + 1])
        a, b = A[s].double(), B[e].double()
        v, mag = a @ b, a.abs() @ b.abs()
        if bias is not None:
            v, mag = v + bias[e].double(), mag + bias[e].double().abs()
        err = act_error(v, sum_error(A.shape[1], mag), act)
        ref[s] = act64(v, act)
        tol[s] = rounded(ref[s], err, A.dtype)
    return ref, tol


def ref_wgrad(A, G, offsets):
    """(reference, bound) of grouped_gemm_wgrad."""
    off = offsets.tolist()
    E = len(off) - 1
    ref = torch.zeros((E, A.shape[1], G.shape[1]), dtype=torch.float64, device=A.device)
    tol = torch.zeros_like(ref)
    for e in range(E):
        a, g = A[off[e]:off[e + 1]].double(), G[off[e]:off[e + 1]].double()
        ref[e] = a.T @ g
        if a.shape[0]:
            tol[e] = rounded(ref[e], sum_error(a.shape[0], a.abs().T @ g.abs()), A.dtype)
    return ref, tol


def ref_lora(x, W, down, up, adapter, scale=None, bias=None, act="none"):
    """(reference, bound) of lora_gemm.

    h is an fp32 sum of K products, scaled (one more rounding of 2^-24); what
    its two 16-bit parts leave out is a quarter step of a step, at most
    half_step^2 of |h|, or half a subnormal step of the type.
    """
    K, R = x.shape[1], down.shape[2]
    dt, xd = x.dtype, x.double()
    v, mag = xd @ W.double(), xd.abs() @ W.double().abs()
    err = torch.zeros_like(v)
    ids = adapter.long()
    for a in ids.unique().tolist():
        if not 0 <= a < down.shape[0]:
            continue
        at = (ids == a).nonzero().flatten()
        s = 1.0 if scale is None else float(scale[a])
        d, u = down[a].double(), up[a].double()
        h, h_mag = s * (xd[at] @ d), abs(s) * (xd[at].abs() @ d.abs())
        tiny = torch.finfo(dt).smallest_normal * half_step(dt)
        h_err = sum_error(K, h_mag) + 2.0 ** -24 * h_mag + half_step(dt) ** 2 * h.abs() + tiny
        v[at] += h @ u
        mag[at] += h.abs() @ u.abs()
        err[at] += h_err @ u.abs()
    if bias is not None:
        v, mag = v + bias.double(), mag + bias.double().abs()
    err = act_error(v, err + sum_error(K + 2 * R, mag), act)
    ref = act64(v, act)
    return ref, rounded(ref, err, dt)
