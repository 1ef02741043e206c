"""Packed prompts long enough for workgroups of 128 pairs whose keys are not split, at both head dimensions, grouped heads, every
cache format and every pair of q's and o's types, against the formula in 64 bits; and a batch served from end to end by a
model of 128 dimensions a head."""
import math
import numpy as np
import pytest
import torch
import seq_cases as S
from test_gpu_20_serving import close
from test_gpu_21_service_bounds import ints, ops

pytestmark = pytest.mark.gpu


def attend(q, values, where, limit, kv, hd, eps):
  """softmax(q k / sqrt(hd)) v in 64 bits for q [L][heads hd], row t over the first limit[t] of cache rows `where`, a key head at
  a time, and a bound of a kernel's error before its output's own rounding: q and the weights in terms off by eps, scores, weights
  and sums in 32 bits (each as in test_gpu_21_service_bounds.attend)."""
  L, heads = q.shape[0], q.shape[1] // hd
  rep, n = heads // kv, len(where)
  q = q.double().view(L, heads, hd)
  out, tol = torch.zeros(L, heads, hd, dtype=torch.float64), torch.zeros(L, heads, hd, dtype=torch.float64)
  hidden = torch.arange(n)[None] >= torch.as_tensor(limit)[:, None]
  for h in range(heads):
    k, v = values[h // rep][where], values[kv + h // rep][where]
    s, size = q[:, h] @ k.T / math.sqrt(hd), q[:, h].abs() @ k.abs().T / math.sqrt(hd)
    p = torch.softmax(s.masked_fill(hidden, -math.inf), 1)
    ds = ((hd + 2) * 2.0 ** -24 * size + eps * size + 8 * 2.0 ** -24 * (1 + s.abs())).masked_fill(hidden, 0).amax(1, keepdim=True)
    out[:, h] = p @ v
    tol[:, h] = (2 * ds + (n + 16) * 2.0 ** -24 + eps) * (p @ v.abs())
  return out.reshape(L, -1), tol.reshape(L, -1)


@pytest.mark.parametrize("fmt", ["bf16", "bfp8", "bfp4", "fp32"])
@pytest.mark.parametrize("q,o", [("bf16", "bf16"), ("fp32", "bf16"), ("bf16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("heads,kv,hd,lens,cached,prefix", [(32, 8, 128, [700, 0, 333], [0, 0, 50], 0), (32, 8, 64, [700, 333, 1], [0, 50, 0], 130),
                                                            (32, 32, 128, [1030], [0], 0)])
def test_long_prompts(cuda, fmt, q, o, heads, kv, hd, lens, cached, prefix):
  print(f"long {lens} {cached} {prefix} {heads}/{kv} {hd} {fmt} {q} {o}", flush=True)
  rng = np.random.default_rng(81)
  n = len(lens)
  first = prefix + 3 + np.concatenate([[0], np.cumsum([a + c + 1 for a, c in zip(lens, cached)])])
  cache, values = S.cache(rng, 2 * kv, int(first[-1]) + 2, hd, fmt)
  qb = torch.from_numpy(rng.normal(0, 0.5, (sum(lens), heads * hd)).astype(np.float32)).to(S.DTYPE[q])
  starts = np.concatenate([[0], np.cumsum(lens)])
  got = ops().attention_prefill_packed(qb.cuda(), cache, heads, kv, hd, ints(starts), ints([prefix + c for c in cached]), ints(first[:-1]),
                                       prefix + max(a + c for a, c in zip(lens, cached)), prefix_row=ints([2]) if prefix else None,
                                       shared=ints([prefix] * n) if prefix else None, out_dtype=S.DTYPE[o]).double().cpu()
  for s, (a, c) in enumerate(zip(lens, cached)):
    lo = int(starts[s])
    # (every third row and the last 40, in 64 bits)
    some = sorted(set(range(0, a, 3)) | set(range(max(0, a - 40), a)))
    if not some: continue
    rows = torch.tensor(some)
    want, tol = attend(qb[lo:lo + a][rows], values, S.rows_of(2, prefix, int(first[s]), prefix + c + a), prefix + c + 1 + np.array(some), kv, hd,
                       2.0 ** -16 if o == "bf16" else 2.0 ** -24)
    err, most = (got[lo:lo + a][rows] - want).abs(), tol + (2.0 ** -8 * (want.abs() + tol) if o == "bf16" else 0) + 1e-30
    assert (err <= most).all(), (s, int((err > most).sum()), float((err / most).max()))


@pytest.mark.parametrize("kv,n", [("bf16", 4), ("bfp8", 4), ("fp32", 2)])
def test_a_batch_of_a_model_with_128_dimensions_a_head(cuda, kv, n):
  # a prefix, packed prompts behind it and steps, against a Decoder that holds every sequence whole (test_gpu_20_serving's bar)
  from ferrite_amd import llama as G
  from oracle import llama as OL
  rng = np.random.default_rng(82)
  cfg = dict(dim=512, heads=8, kv=2, head_dim=128, layers=2, eps=1e-5, theta=10000.0, vocab=1024, ffn=768, places=700)
  w = G.numpy_weights(OL.random_weights(OL.model(**cfg), rng))
  system, prompts = [int(i) for i in rng.integers(0, 1024, 150)], [[int(i) for i in rng.integers(0, 1024, m)] for m in (300, 5, 64, 129)[:n]]
  whole = G.Decoder(G.model(**cfg), w, mode="bfp8", kv=kv, batch=n, context=600, slots=n)
  dec = G.Decoder(G.model(**cfg), None, mode="bfp8", kv=kv, batch=n, context=400, slots=n + 1, share=whole)
  want = torch.cat([whole.prefill(system + p, slot=i)[0].clone() for i, p in enumerate(prompts)])
  dec.prefill(system, slot=n)
  dec.share_prefix(n, 150)
  close(dec.prefill_batch(prompts)[0], want, "prompts' logits")
  places = [150 + len(p) for p in prompts]
  for step in range(2):
    tokens = [int(i) for i in rng.integers(0, 1024, n)]
    close(dec.step(tokens, places, list(range(n)))[0], whole.step(tokens, places, list(range(n)))[0], ("step", step))
    places = [p + 1 for p in places]
