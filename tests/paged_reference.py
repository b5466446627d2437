"""Plain 64-bit forms of the paged cache operators, with elementwise bounds on a kernel's error, and small cases."""
import torch

BF16 = torch.bfloat16
HALF_STEP = 2.0 ** -8  # a rounding to bf16 is off by at most eps / 2 = 2^-8 relative
NAN = float("nan")


def rng(seed):
    return torch.Generator().manual_seed(seed)


class Case:
    """Sequences of the given lengths in shuffled pages. Whatever no sequence holds is NaN: the rows behind a
    sequence's last position, the pages of nobody; table entries past a sequence's pages are far out of range."""

    def __init__(self, lengths, kv_heads, dim, page, seed=0, spare=3, columns=None, one_pool=False, share=0):
        g = rng(seed)
        self.lengths, self.page, self.kv_heads, self.dim = lengths, page, kv_heads, dim
        need = [-(-n // page) for n in lengths]
        total = sum(need) + spare
        order = torch.randperm(total, generator=g)
        columns = max(max(need), 1) if columns is None else columns
        self.table = torch.full((len(lengths), columns), 1 << 30, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n].to(torch.int32)
            at += n
        # `share` leading pages of sequence 0 are those of every other sequence that is long enough, too
        for s, n in enumerate(lengths[1:], 1):
            self.table[s, :min(share, n // page)] = self.table[0, :min(share, n // page)]
        pool = torch.full((total, 2, kv_heads, page, dim), NAN, dtype=BF16)
        for s, n in enumerate(lengths):
            for j in range(need[s]):
                rows = min(page, n - j * page)
                pool[self.table[s, j], :, :, :rows] = torch.randn(2, kv_heads, rows, dim, generator=g).to(BF16)
        self.keys, self.values = (pool[:, 0], pool[:, 1]) if one_pool else (pool[:, 0].clone(), pool[:, 1].clone())

    def to(self, device):
        if self.keys.is_contiguous():
            return self.keys.to(device), self.values.to(device), self.table.to(device)
        pool = torch.stack((self.keys, self.values), 1).to(device)
        return pool[:, 0], pool[:, 1], self.table.to(device)

    def sequence(self, s, length):
        return sequence(self.keys, self.table[s], length), sequence(self.values, self.table[s], length)


def sequence(pool, table, length):
    """[kv_heads, length, dim] in 64 bits."""
    page = pool.shape[2]
    rows = pool[table[:-(-length // page)].long()]                    # [n, heads, page, dim]
    return rows.permute(1, 0, 2, 3).flatten(1, 2)[:, :length].double()


def attend(query, keys, values, scale):
    """(out, bound) of one query row [q_heads, dim] over keys/values [kv_heads, n, dim], in 64 bits.

    bound: the weights' rounding to bf16 and the output's, 2^-8 each; a score's error is at most
    (dim + 16) steps of 2^-23 (sums that may truncate, the scale, the base-2 exponential's argument) of
    |scale| * sum |q k| and of the largest score, and moves every weight by that much relative, numerator and
    denominator both; sums of n weights and products in 32 bits add n * 2^-23 at most (twice)."""
    q_heads, dim = query.shape
    group, n = q_heads // keys.shape[0], keys.shape[1]
    if n == 0:
        return torch.zeros(q_heads, dim, dtype=torch.float64), torch.zeros(q_heads, dim, dtype=torch.float64)
    q = query.double().view(-1, group, dim)
    scores = scale * q @ keys.mT
    weights = torch.softmax(scores, -1)
    out, spread = weights @ values, weights @ values.abs()
    size = (abs(scale) * q.abs() @ keys.abs().mT).amax(-1, keepdim=True) + scores.abs().amax(-1, keepdim=True)
    slack = 2 * (dim + 16) * 2.0 ** -23 * size + 2 * n * 2.0 ** -23
    # the two roundings compound: (1 + 2^-8)^2 - 1
    return out.reshape(q_heads, dim), (HALF_STEP * (1 + HALF_STEP) * (spread + out.abs())
                                       + 2 * slack * spread).reshape(q_heads, dim)


def turn(x, weight, cos, sin, eps):
    """(o, bound) of [rows, heads, dim] bf16 rows: head norm and rotate-half RoPE in 64 bits.

    bound: one rounding to bf16; before it the norm's sum (dim + 8 steps of 2^-24), the reciprocal root and the
    products are off by under (dim / 2 + 16) * 2^-23 relative, of each of the two terms that are added."""
    y, half = x.double(), x.shape[-1] // 2
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = y * c, torch.cat((-y[..., half:], y[..., :half]), -1) * s
    slack = (x.shape[-1] / 2 + 16) * 2.0 ** -23 * (a.abs() + b.abs())
    return a + b, HALF_STEP * ((a + b).abs() + slack) + slack


def tables(count, dim, theta=10000.0):
    angle = torch.arange(count, dtype=torch.float64)[:, None] * theta ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    angle = torch.cat((angle, angle), 1)
    return angle.cos().to(BF16), angle.sin().to(BF16)


def assert_within(got, want, bound, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    off = (got - want).abs() - bound
    assert (off <= 0).all(), f"{what}: off by {((got - want).abs() / bound.clamp(min=1e-300)).max():.3f} of the bound"
