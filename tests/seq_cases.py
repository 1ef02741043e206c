"""What the tests of the packed and shared-prefix attention share: caches of every format with their values, and the
attention in 64 bits with a bound of each output's error."""
import math
import numpy as np
import torch

DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16}


def cache(rng, planes, rows, hd, fmt, device="cuda"):
  """A random KV cache of `fmt` as ops takes it, and its values in float64 [planes][rows][hd]."""
  from ferrite_amd import ops
  if fmt in DTYPE:
    t = torch.from_numpy(rng.normal(0, 1, (planes, rows, hd)).astype(np.float32)).to(DTYPE[fmt])
    return t.to(device), t.double()
  top = rng.integers(124, 129, (planes, rows, hd // 16, 1))
  most = 127 if fmt == "bfp8" else 7
  q = rng.integers(-most, most + 1, (planes, rows, hd // 16, 16))
  values = torch.from_numpy(q * 2.0 ** (top - (133 if fmt == "bfp8" else 129))).reshape(planes, rows, hd)
  m = q.astype(np.int8).view(np.uint8).reshape(-1)
  if fmt == "bfp4": m = (m[0::2] & 15) | (m[1::2] << 4)
  data = torch.from_numpy(np.concatenate([m, top.astype(np.uint8).reshape(-1)]))
  return ops.BfpCache(data.to(device), fmt, planes, rows, hd), values


def attend(q, values, where, limit, kv, hd, o_bf16):
  """softmax(q k / sqrt(hd)) v in 64 bits for q [L][heads hd] (its values as given) over cache rows `where`, row t seeing the
  first limit[t] of them (none: zeros), and a bound of a kernel's error, each output's own:
    scores   a sum of hd products in 32 bits is off by at most (hd + 2) 2^-24 sum |q k|, a product of q's and k's parts by
             at most 2^-22 of it where q, k go in as two bf16 terms or more (a bf16 output's q as two: 2^-16); the exponent's own
             scale and its exp another 8 2^-24 (1 + |s|); each p is off by twice that (its own and the sum's)
    p        rounded to bf16 for a bf16 output: half a step, 2^-8; 2^-22 where it goes in as terms
    sums     of K terms: K 2^-24
    output   rounded to bf16: 2^-8 of itself (half a step)."""
  L, heads = q.shape[0], q.shape[1] // hd
  out, tol = torch.zeros(L, heads, hd, dtype=torch.float64), torch.zeros(L, heads, hd, dtype=torch.float64)
  q = q.double().view(L, heads, hd)
  for h in range(heads):
    g = h // (heads // kv)
    for t in range(L):
      n = int(limit[t])
      if n <= 0: continue
      k, v = values[g][where[:n]], values[kv + g][where[:n]]
      s = (k @ q[t, h]) / math.sqrt(hd)
      p = torch.softmax(s, 0)
      size = (k.abs() @ q[t, h].abs()) / math.sqrt(hd)
      ds = float(((hd + 2) * 2.0 ** -24 * size + (2.0 ** -16 if o_bf16 else 2.0 ** -22) * size + 8 * 2.0 ** -24 * (1 + s.abs())).max())
      rel = 2 * ds + (n + 16) * 2.0 ** -24 + (2.0 ** -8 if o_bf16 else 2.0 ** -22)
      out[t, h] = p @ v
      tol[t, h] = rel * (p @ v.abs()) + (2.0 ** -8 * out[t, h].abs() if o_bf16 else 0) + 1e-30
  return out.reshape(L, -1), tol.reshape(L, -1)


def rows_of(prefix_row, shared, first, n):
  """The cache rows of a sequence's places 0 .. n - 1."""
  p = np.arange(n)
  return torch.from_numpy(np.where(p < shared, prefix_row + p, first + p - shared))


def check(got, want, tol, what):
  bad = (got.double().cpu() - want).abs() > tol
  assert torch.isfinite(got.float()).all() and not bad.any(), (what, int(bad.sum()), float(((got.double().cpu() - want).abs() / tol.clamp(min=1e-30)).max()))
