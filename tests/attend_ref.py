"""Plain 64-bit forms of the attention forms over a cache (csrc/attend.hip) and the error that their kernels may have.

What a kernel rounds: every p to the inputs' 16 bits (u = eps / 2 of its value) and the result once (u again); the rest is fp32 -- D products per
score, N keys per sum, and an exponential and a handful of products with a relative error of a few 2^-24.  With A = sum p |v| over the
seen rows and X = scaling * sum |q| |k| (which bounds a score's rounding, D * 2^-24 * X, and with it p's relative error):
    |error| <= (u + 2 * (D * X + N + 32) * 2^-24) * A + u * |out| + N * 2^-24 * 2^-7 * max |v|      (max over the keys, per dim)
The last term: fp16 p below 2^-14 * 2^-7 of the largest round to a multiple of 2^-24 * 2^-7."""
import torch

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def attend(q, rows_of, scaling):
    """q [B,H,T,D]; rows_of(b, kv_head_of(h), t) -> (k, v) rows [n,D] that the query sees.  Returns (out, bound) [B,T,H,D] fp64 on the CPU."""
    B, H, T, D = q.shape
    out = torch.zeros(B, T, H, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    u, e = U[q.dtype], 2.0 ** -24
    for b in range(B):
        for h in range(H):
            for t in range(T):
                k, v = rows_of(b, h, t)
                if k.shape[0] == 0:
                    continue
                x = q[b, h, t].double()
                s = (k @ x) * scaling
                p = torch.softmax(s, 0)
                o = p @ v
                A = p @ v.abs()
                X = float((k.abs() @ x.abs()).max()) * scaling
                out[b, t, h] = o
                bound[b, t, h] = (u + 2 * (D * X + k.shape[0] + 32) * e) * A + u * o.abs() + k.shape[0] * 2.0 ** -31 * v.abs().amax(0)
    return out, bound


def check(got, ref, bound):
    got = got.double().cpu().view(ref.shape)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(ref), torch.isnan(got)), "NaN in other places"
    assert torch.equal(ref[~fine & ~torch.isnan(ref)], got[~fine & ~torch.isnan(ref)])
    over = ((got - ref).abs() - bound)[fine]
    assert over.numel() == 0 or float(over.max()) <= 0, (float(over.max()), float((got - ref)[fine].abs().max()))


def window_rows(k, v, lens, T, window, sinks, Hkv, H):
    """rows_of() of a window call: k, v [B,Hkv,rows,D] on the CPU in fp64; lens a list of cached rows per request."""
    G = H // Hkv

    def rows_of(b, h, t):
        p = min(lens[b], k.shape[2] - T) + t
        j = torch.arange(max(0, p + 1))
        if window is not None:
            j = j[(j < sinks) | (j > p - window)]
        return k[b, h // G, j], v[b, h // G, j]

    return rows_of


def prefix_rows(kp, vp, k, v, lens, T, Hkv, H):
    G = H // Hkv

    def rows_of(b, h, t):
        p = min(lens[b], k.shape[2] - T) + t
        if p < 0:
            return k[b, 0, :0], v[b, 0, :0]
        return torch.cat([kp[h // G], k[b, h // G, :p + 1]]), torch.cat([vp[h // G], v[b, h // G, :p + 1]])

    return rows_of
