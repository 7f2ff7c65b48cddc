"""Plain 64-bit attention over one sequence and the bounds that the ragged kernels are held to.

With A = sum_j p_j |e_j| per element, S = max_j sum_c |q_c e_jc| D^-1/2 and N entries:

* a score is a float32 sum of D products of bf16 numbers (exact in float32 each): off by at most
  ds = (D + 8) 2^-24 S, the scaling's and the exponent's roundings included in the 8;
* a weight is then off by 2 ds of itself (its own score and those of the sum), by the hardware
  exponential's 2^-22, and is rounded to bf16 for the product, 2^-8;
* float32 sums of N terms, in any order, add N 2^-24 to the weighted sum and as much to the
  weights', and joining partial results a few more roundings, 2^-21;
* the output is rounded to bf16, 2^-8 of itself.

|o - ref| <= 1.02 ((2 ds + 2^-22 + 2^-8 + 2 N 2^-24 + 2^-21) A + 2^-8 |ref|), the 2 % for products
of these.  The log-sum-exp has ds, N 2^-24, 2^-21 and float32's roundings of itself, 2^-22 |lse|.
"""

import torch


def attend(q, e, seen, sink):
    """q [T, H, D], e [N, D] (float64), seen bool [T, N], sink [H] or None -> (o, lse, bound of o, bound of lse)."""
    t, h, d = q.shape
    q, e = q.double(), e.double()
    n = e.shape[0]
    sc = (q.reshape(t * h, d) @ e.t().contiguous()).view(t, h, n) * d ** -0.5
    mag = (q.abs().reshape(t * h, d) @ e.abs().t().contiguous()).view(t, h, n) * d ** -0.5
    sc = torch.where(seen[:, None, :], sc, torch.full_like(sc, float("-inf")))
    mag = torch.where(seen[:, None, :], mag, torch.zeros_like(mag))
    cols = [sc] if sink is None else [sc, sink.double().view(1, h, 1).expand(t, h, 1)]
    z = torch.logsumexp(torch.cat(cols, -1), -1)
    p = torch.where(seen[:, None, :], torch.exp(sc - z[..., None]), torch.zeros_like(sc))
    # entries that a token does not see must not reach it, whatever they hold
    o, a = torch.zeros(t, h, d, dtype=torch.float64, device=q.device), torch.zeros(t, h, d, dtype=torch.float64, device=q.device)
    for i in range(t):
        ev = e[seen[i]]
        pv = p[i][:, seen[i]]
        o[i], a[i] = pv @ ev, pv @ ev.abs()
    ds = (d + 8) * 2.0 ** -24 * (mag.amax(-1) if n else torch.zeros_like(z))[..., None]
    bound = 1.02 * ((2 * ds + 2.0 ** -22 + 2.0 ** -8 + 2 * n * 2.0 ** -24 + 2.0 ** -21) * a + 2.0 ** -8 * o.abs())
    lb = 1.02 * (ds[..., 0] + n * 2.0 ** -24 + 2.0 ** -21 + 2.0 ** -22 * z.abs().nan_to_num(posinf=0))
    return o, z, bound, lb


def check(got_o, got_lse, ref, what):
    o, z, bound, lb = ref
    go, gl = got_o.double(), got_lse.double()
    assert torch.equal(torch.isnan(go), torch.isnan(o)), f"{what}: NaN in other places"
    fine = ~torch.isnan(o)
    err = (go - o).abs()[fine]
    assert bool((err <= bound[fine] + 1e-30).all()), f"{what}: off by {float((err / bound[fine].clamp_min(1e-30)).max()):.2f} of the bound"
    inf = torch.isinf(z)
    assert torch.equal(gl[inf], z[inf]), f"{what}: lse of tokens that see nothing"
    ok = ~inf & ~torch.isnan(z)
    assert bool(((gl - z).abs()[ok] <= lb[ok]).all()), f"{what}: lse off by {float((gl - z).abs()[ok].max()):.2e}"
