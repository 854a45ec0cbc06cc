"""64-bit references and error bounds of the dense attentions and the page tables (torch on the CPU)."""
import torch

U = 2.0 ** -24                                   # half a step of fp32
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E4M3 = torch.float8_e4m3fn


def softmax_product(q, k, v, seen, scale):
    """q [h, n, D], k [h or 1, L, D], v [h or 1, L, Dv] float64, seen [n, L] -> (out, lse, weights @ |v|, largest sum of the
    magnitudes of a seen score's products)."""
    s = torch.matmul(q, k.transpose(1, 2)) * scale
    s = torch.where(seen, s, torch.full_like(s, -torch.inf))
    top = s.amax(2, keepdim=True) if s.shape[2] else s.new_full((*s.shape[:2], 1), -torch.inf)
    p = torch.where(seen, (s - torch.where(top == -torch.inf, 0.0, top)).exp(), 0.0)
    total = p.sum(2, keepdim=True)
    some = total > 0
    w = torch.where(some, p / torch.where(some, total, 1.0), 0.0)
    # a weight of zero takes nothing, whatever stands behind it
    out = torch.matmul(w, torch.where(seen.any(0)[:, None], v, 0.0))
    lse = torch.where(some, top + total.clamp(min=1e-300).log(), -torch.inf)[..., 0]
    mags = torch.where(seen, torch.matmul(q.abs(), k.abs().transpose(1, 2)) * abs(scale), 0.0)
    worst = mags.amax(2) if s.shape[2] else s.new_zeros(s.shape[:2])
    return out, lse, torch.matmul(w, v.abs()), worst


def bounds(out, lse, absv, worst, D, n, dtype, weight_half, floor):
    """(bound of |out error|, of |lse error|). A score is off by D products' worth of fp32 sums, taken at two half steps
    each (the matrix core adds without rounding to nearest), and by its factor: d = (2 D + 4) U worst; a weight by twice that
    (itself and the sum), exp2 and its argument (8 U (1 + |s - m|), |s - m| < 90: 2^-14 where it is that far, and then the weight
    is below 2^-120), its rounding to weight_half, the sums of n by 2 n U; the output is rounded once. floor: what
    weights below the weights' type's normal range lose, relative to the sum, times the largest magnitude."""
    d = (2 * D + 4) * U * worst
    rel = 2 * d + 2 * n * U + 2.0 ** -18
    return absv * (rel + weight_half)[..., None] + out.abs() * HALF[dtype] + floor, d + 2 * n * U + 2.0 ** -20 + lse.abs() * 4 * U


def check(got, lse, ref, D, n, dtype, weight_half, floor=0.0, where=""):
    out64, lse64, absv, worst = ref
    bo, bl = bounds(out64, torch.where(lse64.isfinite(), lse64, 0.0), absv, worst, D, n, dtype, weight_half, floor)
    eo = (got.double() - out64).abs()
    assert bool((eo <= bo + 1e-30).all()), (where, float((eo / (bo + 1e-30)).max()))
    empty = lse64 == -torch.inf
    assert torch.equal(lse == -torch.inf, empty), where
    el = torch.where(empty, 0.0, (lse.double() - lse64).abs())
    assert bool((el <= bl).all()), (where, float((el / bl).max()))


# ------------------------------------------------------------------------------------------------ cache rows
def make_cache(blocks, bs, row, g, spread=0.3, gap=0):
    """[blocks, bs, row] uint8 rows of normal latents (block stride with `gap` rows between blocks)."""
    n = blocks * (bs + gap)
    raw = torch.zeros(n, row, dtype=torch.uint8)
    if row == 576:
        raw[:] = (torch.randn(n, 576, generator=g) * 4).clamp(-448, 448).to(E4M3).view(torch.uint8)
    else:
        lat = torch.randn(n, 4, 128, generator=g) * torch.exp(spread * torch.randn(n, 4, 1, generator=g))
        sc = lat.abs().amax(2, keepdim=True) / 448.0
        raw[:, :512] = (lat / sc).to(E4M3).view(torch.uint8).view(n, 512)
        raw[:, 512:528] = sc.reshape(n, 4).contiguous().view(torch.uint8).view(n, 16)
        raw[:, 528:] = torch.randn(n, 64, generator=g).to(torch.bfloat16).view(torch.uint8).view(n, 128)
    return raw.view(blocks, bs + gap, row)[:, :bs]


def rows64(raw):
    """Cache rows [n, row] as 576 values in 64 bits."""
    if raw.shape[1] == 576:
        return raw.contiguous().view(E4M3).double()
    n = raw.shape[0]
    sc = raw[:, 512:528].contiguous().view(torch.float32).double()
    lat = raw[:, :512].contiguous().view(E4M3).double().view(n, 4, 128) * sc[..., None]
    return torch.cat((lat.view(n, 512), raw[:, 528:].contiguous().view(torch.bfloat16).double()), 1)


# ------------------------------------------------------------------------------------------------ page tables
class Pages:
    """A pool in Python lists."""

    def __init__(self, pages, bs, requests, columns, order=None):
        self.bs, self.W = bs, columns
        self.table = [[] for _ in range(requests)]
        self.lens = [0] * requests
        self.free = list(order if order is not None else range(pages - 1, -1, -1))
        self.missing = 0

    def step(self, new, n):
        new = [max(x, 0) for x in new]
        start, need = [0], 0
        for x in new:
            start.append(start[-1] + x)
        self.missing = 0
        for b, x in enumerate(new):
            want = min(-(-(self.lens[b] + x) // self.bs), self.W)
            for _ in range(max(0, want - len(self.table[b]))):
                if self.free:
                    self.table[b].append(self.free.pop())
                else:
                    self.missing += 1
        req, pos, slot = [], [], []
        for b, x in enumerate(new):
            for i in range(x):
                p = self.lens[b] + i
                c = p // self.bs
                req.append(b)
                pos.append(p)
                slot.append(self.table[b][c] * self.bs + p % self.bs if c < len(self.table[b]) else -1)
        pad = max(0, n - len(req))
        self.lens = [a + x for a, x in zip(self.lens, new)]
        return start, (req + [len(new) - 1] * pad)[:n], (pos + [0] * pad)[:n], (slot + [-1] * pad)[:n]

    def trim(self, keep):
        back = []
        for b, k in enumerate(keep):
            self.lens[b] = min(self.lens[b], max(k, 0))
            left = -(-self.lens[b] // self.bs)
            back += self.table[b][left:]
            del self.table[b][left:]
        self.free += back[::-1]

    def same_as(self, pool):
        t = pool.table.cpu().tolist()
        want = [r + [-1] * (self.W - len(r)) for r in self.table]
        assert t == want
        assert pool.lens.cpu().tolist() == self.lens and pool.held.cpu().tolist() == [len(r) for r in self.table]
        n = len(self.free)
        assert pool.state.cpu().tolist()[:3] == [n, self.missing, 0] and pool.free.cpu().tolist()[:n] == self.free
