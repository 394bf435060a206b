"""Plain 64-bit forms of the attention operators and how far the kernels may be off them.

Bounds.  With w_j the softmax weights and A = sum_j w_j |v_j|: rounding the output to bf16 is off by at most 2^-8 of it;
rounding each weight before the product with V (bf16: 2^-8, f16: 2^-11 of the weight, and 2^-32 of the largest weight
where it is subnormal in f16: half a step, 2^-25, of weights the largest of which is taken as 2^7 or more) moves the output by at most that share of A; a score off by d changes every weight by at
most a factor exp(2 d).  Scores are fp32 sums of D products: each of the D additions and the scaling rounds by 2^-24 of
at most S = max scale sum |q_d k_d|, and 2^x of the hardware is good to 2^-22, the sums of the weights to 2^-20.
"""
import math

import torch


def visible(nq, nk, left, right, sinks, device):
    p = torch.arange(nq, device=device)[:, None] + (nk - nq)
    j = torch.arange(nk, device=device)[None, :]
    see = torch.ones(nq, nk, dtype=torch.bool, device=device)
    if right >= 0:
        see &= j <= p + right
    if left >= 0:
        see &= (j >= p - left) | (j < sinks)
    return see


def attention_rows(q, k, v, scale, see, weight_step=2.0 ** -8, weight_floor=0.0):
    """q [n, D], k and v [m, D] (any float type) -> (out, lse, bound of out, bound of lse) in float64."""
    q, k, v = q.double(), k.double(), v.double()
    D = q.shape[1]
    k, v = torch.where(see.any(0)[:, None], k, 0), torch.where(see.any(0)[:, None], v, 0)  # what nobody sees may hold anything
    s = torch.where(see, scale * (q @ k.T), -math.inf)
    m = s.amax(1, keepdim=True) if s.shape[1] else torch.full((q.shape[0], 1), -math.inf, dtype=torch.float64, device=q.device)
    e = torch.exp(s - torch.where(m.isinf(), 0, m))
    total = e.sum(1, keepdim=True)
    w = e / total.clamp(min=1e-300)
    out, lse = w @ v, (m + total.log())[:, 0]
    size = torch.where(see, scale * (q.abs() @ k.abs().T), 0).amax(1, keepdim=True) if s.shape[1] else torch.zeros_like(m)
    off = (D + 4) * 2.0 ** -24 * size + 2.0 ** -20
    spread = w @ v.abs()
    few = weight_floor * see.double() @ v.abs()
    bound = 2.0 ** -8 * out.abs() + (weight_step + 2 * off) * (1 + 2.0 ** -8) * spread + few + 1e-30
    return out, lse, bound, off[:, 0] + 2.0 ** -23 * lse.abs().nan_to_num(posinf=0)


def window_reference(q, k, v, rows, keys, H, Hkv, D, scale, left, right, sinks):
    """q [sum(rows), H, D], k and v [sum(keys), Hkv, D], sequences one behind the other."""
    outs = [torch.zeros(q.shape[0], H, D, dtype=torch.float64, device=q.device) for _ in range(2)]
    lses = [torch.zeros(q.shape[0], H, dtype=torch.float64, device=q.device) for _ in range(2)]
    i = j = 0
    for nq, nk in zip(rows, keys):
        see = visible(nq, nk, left, right, sinks, q.device)
        for h in range(H):
            g = h // (H // Hkv)
            o, l, bo, bl = attention_rows(q[i:i + nq, h], k[j:j + nk, g], v[j:j + nk, g], scale, see)
            outs[0][i:i + nq, h], outs[1][i:i + nq, h], lses[0][i:i + nq, h], lses[1][i:i + nq, h] = o, bo, l, bl
        i, j = i + nq, j + nk
    return outs[0], lses[0], outs[1], lses[1]


def gather(t, table, n):
    """The first n tokens [n, Hkv, D] of a sequence out of pages [pages, page_size, Hkv, D], in 64 bits."""
    page = t.shape[1]
    j = torch.arange(n, device=t.device)
    raw = t.view(torch.uint8) if t.dtype.itemsize == 1 else t
    return raw[table.long()[j // page], j % page].view(t.dtype).double()


def decode_reference(q, cache, lens, H, scale, left, sinks):
    """q [n_seqs, H, D] -> (out, lse, bounds)."""
    n, _, D = q.shape
    Hkv = cache.k.shape[2]
    e4m3 = cache.k.dtype != torch.bfloat16
    outs = [torch.zeros(n, H, D, dtype=torch.float64, device=q.device) for _ in range(2)]
    lses = [torch.zeros(n, H, dtype=torch.float64, device=q.device) for _ in range(2)]
    for b, L in enumerate(lens):
        k, v = gather(cache.k, cache.page_table[b], L), gather(cache.v, cache.page_table[b], L)
        see = visible(1, L, left, 0, sinks, q.device)
        for h in range(H):
            g = h // (H // Hkv)
            ks, vs = (1.0 if s is None else float(s[g]) for s in (cache.k_scale, cache.v_scale))
            o, l, bo, bl = attention_rows(q[b, h][None], k[:, g] * ks, v[:, g] * vs, scale, see, 2.0 ** -11 if e4m3 else 2.0 ** -8,
                                          2.0 ** -32 if e4m3 else 0.0)
            outs[0][b, h], outs[1][b, h], lses[0][b, h], lses[1][b, h] = o[0], bo[0], l[0], bl[0]
    return outs[0], lses[0], outs[1], lses[1]


def assert_within(got, want, bound, what=""):
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()]), f"{what}: infinities in other places"
    over = ((got - want).abs() - bound)[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, \
        f"{what}: {int((over > 0).sum())} of {over.numel()} beyond their bound, worst {float(((got - want).abs() / bound)[fin].max()):.2f} of it"


def rope_reference(x, w, cos, sin, rot, mode, eps):
    """x [rows, heads, D] -> 64-bit norm (w None: none) and rotation; cos, sin [rows, rot / 2]; mode 0 none, 1 adjacent pairs, 2 halves."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if mode == 0 or rot == 0:
        return x
    c, s = cos.double()[:, None], sin.double()[:, None]
    y = x.clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if mode == 1 else (x[..., :rot // 2], x[..., rot // 2:rot])
    if mode == 1:
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    else:
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, a * s + b * c
    return y
