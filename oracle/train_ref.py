"""Oracle of the training operators (lbm_amd/training.py): the dropout mask's definition in integer arithmetic on the CPU, and layer
normalisation with its gradients in float64 from the formulas."""
import numpy as np
import torch

M32 = np.uint64(0xFFFFFFFF)
S32 = np.uint64(32)


def philox4x32(counter, key, rounds=10):
    """Philox4x32 (Salmon et al., SC 2011).  counter: four arrays of 32-bit words; key: two words -> four uint64 arrays of 32-bit words."""
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> S32) ^ c[1] ^ np.uint64(k0), b & M32, (a >> S32) ^ c[3] ^ np.uint64(k1), a & M32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def numbers(first, count, seed, offset):
    """The 32-bit numbers of elements first .. first + count - 1."""
    seed, offset = seed % (1 << 64), offset % (1 << 64)
    b0, b1 = first // 8, (first + count + 7) // 8
    blocks = np.arange(b0, b1, dtype=np.uint64)
    halves = []
    for part in (0, 1):
        n = blocks * np.uint64(2) + np.uint64(part)
        full = np.ones_like(n)
        w = philox4x32([n & M32, n >> S32, full * np.uint64(offset & 0xFFFFFFFF), full * np.uint64(offset >> 32)], (seed & 0xFFFFFFFF, seed >> 32))
        halves.append(np.stack([(w[j >> 1] >> np.uint64(16 * (j & 1))) & np.uint64(0xFFFF) for j in range(8)], 1).reshape(-1))
    r = (halves[0] << np.uint64(16)) | halves[1]
    return r[first - 8 * b0:first - 8 * b0 + count]


def keep(shape, p, seed, offset, first=0):
    """Truth values: which elements of a tensor of this shape are kept."""
    n = int(np.prod(shape))
    if n == 0:
        return torch.zeros(shape, dtype=torch.bool)
    return torch.from_numpy(numbers(first, n, seed, offset) >= np.uint64(round(p * 2 ** 32))).reshape(shape)


def scale(p):
    t = round(p * 2 ** 32)
    return 0.0 if t >= 2 ** 32 else 2 ** 32 / (2 ** 32 - t)


def norm(x, weight, bias, eps, residual=None, factor=None, dy=None):
    """float64 forward and gradients; factor = scale where kept, 0 elsewhere (None: nothing dropped).  A dict, with the intermediate
    values that error bounds are made of."""
    x = x.detach().double().cpu()
    xs = x if factor is None else torch.where(factor != 0, x * factor, torch.zeros((), dtype=torch.float64))
    z = xs if residual is None else residual.detach().double().cpu() + xs
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    b = torch.zeros(x.shape[-1], dtype=torch.float64) if bias is None else bias.detach().double().cpu()
    mean = z.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((z - mean) ** 2).mean(-1, keepdim=True) + eps)
    xhat = (z - mean) * rstd
    out = dict(xs=xs, z=z, w=w, b=b, mean=mean, rstd=rstd, xhat=xhat, y=xhat * w + b)
    if dy is not None:
        dy = dy.detach().double().cpu()
        g = dy * w
        c1, c2 = g.mean(-1, keepdim=True), (g * xhat).mean(-1, keepdim=True)
        dz = rstd * (g - c1 - xhat * c2)
        rows = tuple(range(dy.dim() - 1))
        out.update(dy=dy, g=g, c1=c1, c2=c2, dresidual=dz, dx=dz if factor is None else dz * factor,
                   dweight=(dy * xhat).sum(rows) if rows else dy * xhat, dbias=dy.sum(rows) if rows else dy)
    return out
