"""Plain forms of the paged cache's operators in 64 bits, and how far 32 and 16 bits may be from them."""
import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8  # half a step of float32 and of bfloat16, relative


class Pages:
    """The book of pages in lists."""

    def __init__(self, pages, page_size, requests, most):
        self.P, self.most, self.free = page_size, most, list(range(pages))
        self.tables, self.lens = [[] for _ in range(requests)], [0] * requests

    def step(self, new, rows):
        """(row_start, pos, places), or None where the step has no room; the lists are then as before."""
        P = self.P
        want = [max(0, -(-(l + max(n, 0)) // P) - -(-l // P)) for l, n in zip(self.lens, new)]
        if (sum(want) > len(self.free) or sum(max(n, 0) for n in new) > rows
                or any(l + max(n, 0) > P * self.most for l, n in zip(self.lens, new))):
            return None
        taken, row_start, pos, places = self.free[:sum(want)], [0], [], []
        self.free = self.free[sum(want):]
        for i, n in enumerate(new):
            if n < 0:
                self.free += self.tables[i]
                self.tables[i], self.lens[i] = [], 0
            else:
                self.tables[i] = self.tables[i] + taken[:want[i]]
                taken = taken[want[i]:]
                for t in range(self.lens[i], self.lens[i] + n):
                    pos.append(t)
                    places.append(self.tables[i][t // P] * P + t % P)
                self.lens[i] += n
            row_start.append(len(pos))
        return row_start, pos + [0] * (rows - len(pos)), places + [-1] * (rows - len(places))


def attention(q, k, v, see, scale, bits16):
    """Rows q [rows, heads, d] over the first see[r] of the keys k [keys, kv_heads, d] -> ([rows, heads, e], tolerance of each value).

    The tolerance of o = sum p v / sum p: a score's d products and their sum are off by at most (d + 1) U32 sum |q k| scale, the exponent's
    argument by |score| U32 more, its result by a few steps, and these count in numerator and denominator; the two sums add
    keys U32 each. In 16 bits p is rounded once (both sums may differ by that) and the result once. All relative to sum p |v| / sum p."""
    q, k, v = q.double(), k.double(), v.double()
    H, G = q.shape[1], k.shape[1]
    k, v = k.repeat_interleave(H // G, 1), v.repeat_interleave(H // G, 1)
    z = torch.einsum("rhd,khd->rhk", q, k) * scale
    size = torch.einsum("rhd,khd->rhk", q.abs(), k.abs()) * abs(scale)
    hidden = torch.arange(k.shape[0], device=q.device)[None, None] >= see[:, None, None]
    p = torch.softmax(z.masked_fill(hidden, float("-inf")), -1)
    p = torch.where(hidden, 0.0, p)  # a row that sees nothing
    size = torch.where(hidden, 0.0, size).amax(-1, keepdim=True) if k.shape[0] else torch.zeros_like(p.sum(-1, keepdim=True))
    v = torch.nan_to_num(v, nan=0.0, posinf=0.0, neginf=0.0)
    o, a = torch.einsum("rhk,khe->rhe", p, v), torch.einsum("rhk,khe->rhe", p, v.abs())
    steps = 2 * (q.shape[2] + 3) * size + 2 * see.clamp(min=0)[:, None, None] + 32
    return o, a * (steps * U32 + (3 * U16 if bits16 else 0)) + 1e-30


def write(x, H, G, D, V, q_norm, k_norm, pos, vmix, v_first, coef, every, eps=1e-6):
    """(q [rows, H, D], k [rows, G, D], v [rows, G, V]) of projected rows."""
    x = x.double()
    q, k, v = x.split([H * D, G * D, G * V], 1)
    norm = lambda t, w: t.view(x.shape[0], -1, D) / torch.sqrt((t.view(x.shape[0], -1, D) ** 2).mean(-1, keepdim=True) + eps) * w.double()
    t = 1 + coef * torch.log(torch.div(pos + 1, every, rounding_mode="floor").double() + 1) if every else torch.ones_like(pos).double()
    if vmix is not None:
        v = (1 - vmix.double()) * v + vmix.double() * v_first.double().view(v.shape)
    return norm(q, q_norm) * t[:, None, None], norm(k, k_norm), v.reshape(-1, G, V)
