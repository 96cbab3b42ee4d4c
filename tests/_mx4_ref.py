"""Plain 64-bit statements of the microscaled 4-bit format and of the Newton-Schulz iteration (test infrastructure)."""
import numpy as np
import torch

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
NS = (3.4445, -4.7750, 2.0315)


def round_codes(x):
    """x [R,K] float64 -> (codes [R,Kp] 0 ... 15, scale codes [R,Kp/32] 0 ... 255), Kp = K rounded up to 256."""
    x = np.asarray(x, np.float64)
    R, K = x.shape
    kp = -(-K // 256) * 256
    pad = np.zeros((R, kp))
    pad[:, :K] = x
    b = pad.reshape(R, kp // 32, 32)
    with np.errstate(all="ignore"):
        top = np.abs(b).max(axis=2)
        bad = ~np.isfinite(top)
        s = np.where(top > 0, np.frexp(np.where(bad, 1.0, top))[1] - 3, -127)       # floor(log2) - 2
        s = np.clip(s, -127, 127)
        mag = np.abs(np.ldexp(b, -s[..., None]))
        mag = np.where(bad[..., None], 0.0, np.minimum(mag, 6.0))
    d = np.abs(mag[..., None] - LEVELS)
    # nearest; of two equally near ones the even code
    near = d == d.min(axis=-1, keepdims=True)
    code = np.where(near.sum(-1) == 2, np.where(near[..., 0::2].any(-1), 2 * near[..., 0::2].argmax(-1), near.argmax(-1)),
                    near.argmax(-1))
    code = code + 8 * (np.signbit(b) & ~bad[..., None])
    return code.reshape(R, kp), np.where(bad, 255, s + 127).reshape(R, kp // 32)


def code_values(codes, scales, K):
    lev = LEVELS[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    R, kp = codes.shape
    with np.errstate(all="ignore"):
        s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales - 127))
    return (lev.reshape(R, kp // 32, 32) * s[..., None]).reshape(R, kp)[:, :K]


def values(x):
    """The rounded values of x [R,K] (a tensor) in float64."""
    a = x.detach().double().cpu().numpy()
    return torch.from_numpy(code_values(*round_codes(a), a.shape[1]))


def unpack(q):
    """(codes [R,Kp], scales) of an Mx4Tensor."""
    c = q.codes.cpu().numpy()
    out = np.empty((c.shape[0], 2 * c.shape[1]), np.int64)
    out[:, 0::2], out[:, 1::2] = c & 15, c >> 4
    return out, q.scales.cpu().numpy().astype(np.int64)


def orthogonal(g, steps=5, eps=1e-7, dtype=torch.float64):
    x = g.detach().cpu().to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.norm() + eps)
    for _ in range(steps):
        s = x @ x.t()
        x = NS[0] * x + (NS[1] * s + NS[2] * (s @ s)) @ x
    return x.t() if tall else x
