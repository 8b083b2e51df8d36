"""Plain 64-bit forms of the 4-bit and expert operators, for their tests
(numpy, written from the definitions in include/xse_mx.h and
include/xse_experts.h)."""

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MIDDLE = (GRID[1:] + GRID[:-1]) / 2


def quantize(x):
  """(codes [rows, padded], scale bytes [rows, blocks]) of x [rows, cols]."""
  x = np.asarray(x, np.float64)
  rows, cols = x.shape
  blocks = -(-cols // 32)
  v = np.zeros((rows, blocks * 32))
  v[:, :cols] = x
  v = v.reshape(rows, blocks, 32)
  bad = ~np.isfinite(v).all(axis=2)
  v = np.where(bad[..., None], 0.0, v)
  most = np.abs(v).max(axis=2)
  _, e = np.frexp(most)  # most = m 2^e, 0.5 <= m < 1
  s = np.where(most > 0, np.maximum(e - 1 - 2, -127), -127) + 127
  a = np.abs(v) / np.exp2(s - 127.0)[..., None]
  code = np.zeros(a.shape, np.int64)
  for k in range(7):  # a tie goes to the even one of codes k and k + 1
    code += (a > MIDDLE[k]) if k % 2 == 0 else (a >= MIDDLE[k])
  code += 8 * np.signbit(v)
  code[bad] = 0
  s = np.where(bad, 255, s)
  return code.reshape(rows, blocks * 32), s.astype(np.int64)


def values(codes, s, cols):
  """The values codes and scale bytes stand for, [rows, cols]."""
  rows = codes.shape[0]
  v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
  scale = np.where(s == 255, np.nan, np.exp2(s - 127.0))
  v = v.reshape(rows, -1, 32) * scale[..., None]
  return v.reshape(rows, -1)[:, :cols]


def quantized(x):
  codes, s = quantize(x)
  return values(codes, s, x.shape[1])


def pack_codes(codes):
  return (codes[:, 0::2] & 15 | (codes[:, 1::2] & 15) << 4).astype(np.uint8)


def scale_offsets(rows, blocks):
  """Byte offset of each block's scale in its group's tiles."""
  k_tiles = -(-blocks // 4)
  r = np.arange(rows)[:, None]
  b = np.arange(blocks)[None, :]
  return ((r // 128) * k_tiles + b // 4) * 512 + r % 32 * 16 + \
      r % 128 // 32 * 4 + b % 4


def activate(y, act):
  if act == 1:
    return np.where(y < 0, 0.0, y)
  if act == 2:
    return 1.0 / (1.0 + np.exp(-np.clip(y, -700.0, 700.0)))
  return y


def linear(x, w, bias, act):
  """(act(Q(x) w^T + bias), sum |Q(x)||w|^T + |bias|) for w's own values."""
  q = quantized(x)
  y, size = q @ w.T, np.abs(q) @ np.abs(w).T
  if bias is not None:
    y, size = y + bias, size + np.abs(bias)
  return activate(y, act), size


def linear_tolerance(y, size, k, eps):
  """The products are exact in fp32 (four significant bits and a power of
  two). Adding k of them and the bias one after another is off by at most one
  unit of the last place (2^-23, truncation) of the sum of magnitudes an
  addition; activations do not enlarge that, a sigmoid's own error is a few
  units; the result is rounded once to a type of spacing eps."""
  return (k + 8) * 2.0 ** -23 * (size + 1e-30) + eps / 2 * np.abs(y) + 1e-38


def sort(ids, experts):
  """offsets, order, slots of ids [tokens, topk]."""
  flat = np.asarray(ids).reshape(-1)
  by = [np.nonzero(flat == e)[0] for e in range(experts)]
  offsets = np.concatenate([[0], np.cumsum([len(b) for b in by])])
  order = np.full(flat.size, -1)
  kept = np.concatenate(by) if by else np.zeros(0, np.int64)
  order[:kept.size] = kept
  slots = np.full(flat.size, -1)
  slots[kept] = np.arange(kept.size)
  return offsets, order, slots.reshape(np.shape(ids))
