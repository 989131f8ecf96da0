"""Data on which every cached position shows: position j of n has the value 1 in column j * hd // n and 0 elsewhere, and a
key whose element 0 is 0 where it counts (every `step`-th position) and so low elsewhere that its weight is 0.  With a
query of (1, 0, ..) the result of a column is the number of its positions that count over the number of all that do: sums
of ones are exact, so a kernel may be off by the division and the product with it, and a position that is left out or
counted twice moves its column by one in n / hd / step."""
import torch

SLACK = 2.0 ** -22


def low(dtype):
    """A score whose weight is 0 in float32 and that the type holds."""
    return -448.0 if dtype == torch.float8_e4m3fn else -1000.0


def rows(n, hd, step, dtype, seed):
    """Keys and values [n, hd] of one sequence; the keys' other elements are noise that the query does not see."""
    g = torch.Generator().manual_seed(seed)
    j = torch.arange(n)
    k, v = torch.randn(n, hd, generator=g), torch.zeros(n, hd)
    k[:, 0] = torch.where(j % step == 0, 0.0, low(dtype))
    v[j, j * hd // max(n, 1)] = 1.0
    return k.to(dtype), v.to(dtype)


def result(n, hd, step, used=None, of=None):
    """What the columns of a sequence's result are when it has `used` of the positions of rows(of or n, ..) (default: the
    first n)."""
    j = torch.arange(n) if used is None else used
    j = j[j % step == 0]
    count = torch.bincount(j * hd // max(of or n, 1), minlength=hd).double()
    return count / count.sum() if len(j) else count
