"""Reference and error bound for the attention of packed sequences, shared by its tests.

attend64: out[t, h] = sum_{u <= t} softmax_u(scale q[t, h] . k[u, kv]) v[u, kv] in 64 bits, for one sequence whose
n queries are its last n tokens; keys with there[u] False are not attended to.

Bound per element, with EPS = 2^-24 and u = half a step of the type (2^-11 for fp16, 2^-8 for bf16):
* a score is a 32-bit sum of d exact products, scaled and subtracted in the exponent: (d + 8) EPS of
  sum |q k| scale absolute error, hence twice that as a relative error of a probability over the sum of them;
* the hardware exponential, the sums over n keys, the joins of partial sums and the division: (n + 64) EPS;
* the probability is rounded for the second product: u, or in fp16 below 2^-14 at most 2^-25 of a largest probability
  that is at least 1 (the exponentials are taken against a maximum that was reached): 2^-25 sum |v|;
* the result is rounded: u (and half of the type's smallest step).
"""

from __future__ import annotations

import math

import torch

EPS = 2.0 ** -24
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend64(q, k, v, there=None, scale=None):
    """(reference, bound) float64 [n, heads, d] for q [n, heads, d] and k, v [keys, kv_heads, d]."""
    n, heads, d = q.shape
    keys, kv_heads, _ = k.shape
    rep = heads // kv_heads
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    u = HALF_STEP[q.dtype]
    first = keys - n
    seen = torch.arange(keys, device=q.device)[None, :] <= (first + torch.arange(n, device=q.device))[:, None]
    if there is not None:
        seen = seen & there[None, :]
    ref = torch.zeros(n, heads, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(ref)
    for h in range(heads):
        q64, k64, v64 = q[:, h].double(), k[:, h // rep].double(), v[:, h // rep].double()
        s = torch.where(seen, (q64 @ k64.T) * scale, -math.inf)
        top = s.amax(-1, keepdim=True) if keys else s.new_full((n, 1), -math.inf)
        p = torch.where(seen, torch.exp(s - torch.where(top.isinf(), 0.0, top)), 0.0)
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        # A key that no row attends to adds nothing, whatever its value is.
        v_seen = torch.where(seen.any(0)[:, None], v64, 0.0)
        ref[:, h] = p @ v_seen
        mag = torch.where(seen, (q64.abs() @ k64.abs().T) * scale, 0.0).amax(-1, keepdim=True) if keys else 0.0
        rel = u + 2 * (d + 8) * EPS * mag + (keys + 64) * EPS
        sub = 2.0 ** -25 * (seen.double() @ v_seen.abs()) if q.dtype == torch.float16 else 0.0
        bound[:, h] = rel * (p @ v_seen.abs()) + sub + u * ref[:, h].abs() + 2.0 ** -25
    return ref, bound


def check(out, ref, bound, what=""):
    err = (out.double() - ref).abs()
    assert out.isfinite().all(), f"{what}: not finite"
    worst = float((err / bound).max()) if out.numel() else 0.0
    assert worst <= 1.0, f"{what}: largest error / bound {worst:.2f}"
    return worst


def offsets(lens, device):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=device)
