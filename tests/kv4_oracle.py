"""The 4-bit cache's formulas in 64 bits: what stored rows are worth, attention over them with its error bound, eviction."""
import torch


def stored(x):
    """What bf16 rows x [..., d] are worth once stored: per 64 columns code * step + lowest, the step a bf16 number not below
    (max - min) / 15."""
    v = x.double().cpu().unflatten(-1, (-1, 64))
    lo, hi = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
    rng = hi - lo
    rng = torch.where(rng.float().isfinite(), rng, torch.full_like(rng, float("nan")))
    step = rng / 15
    e = torch.floor(torch.log2(step.clamp_min(1e-300))).clamp_min(-126)
    unit = torch.exp2(e - 7)
    step = torch.ceil(step / unit) * unit
    code = torch.where(step > 0, torch.round((v - lo) / torch.where(step > 0, step, torch.ones_like(step))).clamp(0, 15), torch.zeros_like(v))
    return (code * step + lo).flatten(-2), step.squeeze(-1), lo.squeeze(-1)


def attention(q, k, v, scale, k_step, k_low, v_step, v_low):
    """q [r, d], k, v [n, d] (64 bits) -> out, weights p, and what fp32 sums and 16-bit products may be off by: the relative error of the
    weights, sum p |v|, and an absolute error of the result.

    Scores.  A kernel may multiply q by codes with an offset of up to 64 and take the offset off in the sum, and add q lowest: an fp32 sum
    of d products has an error of at most (d + 16) 2^-24 sum_i |q_i| ((64 + 15 + 64) step_i + |lowest_i|) scale =: e.  A weight
    p = exp(s) / sum exp is then off by a factor of at most exp(2 e), and by 2^-20 more for its exponentials (2^-22 each) and sums.
    Values.  With mid = lowest + 8 step, step p may be rounded to fp16 (half a step is 2^-11 of it) ahead of its product with code - 8, while
    sum p mid is carried in fp32: an error of at most 2^-11 sum_t p_t |v_t - mid_t|.  Both are fp32 sums of n terms, a few multiplications and
    additions more: (n + 16) 2^-24 sum_t p_t (|v_t - mid_t| + |mid_t|), which is not small against v where it is far below mid.  The fp16
    numbers are step p 128 / M, with M at most twice the largest step and the largest p at least 1 ahead of the division by sum p: below their
    smallest they are off by 2^-25, which 8 M / 128 multiplies: 2^-28 max step for each of the n tokens at most."""
    s = q.double() @ k.T * scale
    p = torch.softmax(s, -1)
    d = q.shape[-1]
    mag = (143 * k_step + k_low.abs()).repeat_interleave(64, -1)
    e = ((d + 16) * 2.0 ** -24 * abs(scale) * (q.double().abs() @ mag.T)).amax(-1, keepdim=True)
    rel = torch.expm1(2 * e) + 2.0 ** -20
    mid = (v_low + 8 * v_step).repeat_interleave(64, -1)
    far = (v - mid).abs()
    return p @ v, p, rel, p @ v.abs(), 2.0 ** -11 * (p @ far) + (len(v) + 16) * 2.0 ** -24 * (p @ (far + mid.abs())) \
        + len(v) * 2.0 ** -28 * v_step.amax(0).repeat_interleave(64, -1)


def keep(weights, positions, n, seen, budget, first, last):
    """One request and head: lists of n weights and positions -> the place whose token each place below min(n, budget) holds."""
    if n <= budget:
        return list(range(n))

    def rank(j):
        if positions[j] < first or positions[j] >= seen - last:
            return (0, 0.0, j)
        return (1, 0.0, j) if weights[j] != weights[j] else (2, -weights[j], j)
    stay = sorted(sorted(range(n), key=rank)[:budget])
    inside = set(j for j in stay if j < budget)
    outside = [j for j in stay if j >= budget]
    return [j if j in inside else outside.pop(0) for j in range(budget)]
