"""What a batch's calls keep to where they could go wrong unseen: attention's bf16 output within its own rounding and the 2^-16
that its weights and q are held to; heads under grammars that leave whole parts of a row empty; rows given on the GPU; one
workspace for a service's largest calls."""
import math
import numpy as np
import pytest
import torch
import seq_cases as S
from oracle.serve import head_of

pytestmark = pytest.mark.gpu


def ops():
  from ferrite_amd import ops as m
  return m


def ints(v):
  return torch.tensor(list(v), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("V", [49152, 4100, 128256])
def test_heads_under_a_mask_that_leaves_parts_of_a_row_empty(cuda, V):
  # a grammar that allows a few columns of one part of 4096, one that allows columns of the last part alone, none at all, all
  rng = np.random.default_rng(V)
  x = rng.normal(0, 3, (4, V)).astype(np.float32)
  bits = np.zeros((4, V), bool)
  bits[0, 11:60], bits[1, V - 3:], bits[3] = True, True, True
  words = np.zeros((4, -(-V // 32) * 32), np.uint32)
  words[:, :V] = bits
  words = (words.reshape(4, -1, 32) << np.arange(32, dtype=np.uint32)).sum(2, dtype=np.uint32).view(np.int32)
  y = ops().logit_rules(torch.from_numpy(x).cuda(), allowed=torch.from_numpy(words).cuda())
  t = [1.0, 0.5, 2.0, 1 / 0.7]
  values, ids, lse = ops().logit_heads(y, 40, torch.tensor(t, dtype=torch.float32, device="cuda"))
  z = np.where(bits, x, -np.inf).astype(np.float32)
  for r in (0, 1, 3):
    wv, wi, wl = head_of(z[r], float(np.float32(t[r])), 40)
    assert np.array_equal(ids[r].cpu().numpy(), wi) and np.array_equal(values[r].cpu().numpy(), wv), r
    # (fp32: the maximum's product, each exp and its argument, a sum of at most V terms pairwise, the log: test_heads' bound)
    assert abs(float(lse[r]) - wl) <= 2e-6 * abs(wl) + 2e-6, (r, float(lse[r]), wl)
  # (nothing left: no sum, the first columns, -inf each)
  assert float(lse[2]) == -math.inf and (values[2] == -math.inf).all() and ids[2].tolist() == list(range(40))


def attend(q, values, where, limit, kv, hd):
  """softmax(q k / sqrt(hd)) v in 64 bits for q [L][heads hd], row t over the first limit[t] of cache rows `where`, and a bound
  of a kernel's error before its output's own rounding: scores in 32 bits (a sum of hd products: (hd + 2) 2^-24 of the sum of
  their sizes, and 2^-16 of it for q in two bf16 terms; the exponent's scale and exp 8 2^-24 (1 + |s|)), twice that for
  each weight (its own and the sum's), the weights in two bf16 terms 2^-16, sums of n terms n 2^-24."""
  L, heads = q.shape[0], q.shape[1] // hd
  rep = heads // kv
  q = q.double().view(L, kv, rep, hd).transpose(0, 1)                                   # [kv][L][rep][hd]
  k, v = values[:kv][:, where], values[kv:][:, where]                                   # [kv][n][hd]
  s = torch.einsum("glrd,gnd->glrn", q, k) / math.sqrt(hd)
  size = torch.einsum("glrd,gnd->glrn", q.abs(), k.abs()) / math.sqrt(hd)
  seen = (torch.arange(len(where))[None] < torch.as_tensor(limit)[:, None])[None, :, None]
  p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
  out, big = torch.einsum("glrn,gnd->glrd", p, v), torch.einsum("glrn,gnd->glrd", p, v.abs())
  ds = ((hd + 2) * 2.0 ** -24 * size + 2.0 ** -16 * size + 8 * 2.0 ** -24 * (1 + s.abs())).masked_fill(~seen, 0).amax(-1, keepdim=True)
  tol = (2 * ds + (len(where) + 16) * 2.0 ** -24 + 2.0 ** -16) * big
  return (t.transpose(0, 1).reshape(L, heads * hd) for t in (out, tol))


def check(got, want, tol, what):
  # (bf16: half a step of what the kernel holds, 2^-8 of it)
  err = (got.double().cpu() - want).abs()
  most = tol + 2.0 ** -8 * (want.abs() + tol) + 1e-30
  assert (err <= most).all(), (what, int((err > most).sum()), float((err / most).max()))


HEADS = [(9, 3, 64, "bf16", "fp32"), (8, 2, 128, "bfp8", "fp32"), (8, 2, 128, "bf16", "bf16"), (4, 4, 64, "bfp4", "bf16"), (32, 8, 128, "bf16", "fp32")]


@pytest.mark.parametrize("heads,kv,hd,fmt,q", HEADS)
@pytest.mark.parametrize("lens,cached", [([20, 1, 33], [0, 40, 7]), ([300, 150], [0, 90]), ([2, 3], [700, 900])])
def test_packed_bf16_output(cuda, heads, kv, hd, fmt, q, lens, cached):
  # (scores near 0, so that the bound is of the weights' rounding and not the scores')
  print(f"packed bf16 {lens} {cached} {heads}/{kv} {hd} {fmt} {q}", flush=True)
  rng = np.random.default_rng(71)
  first = np.concatenate([[2], 2 + np.cumsum([a + c + 1 for a, c in zip(lens, cached)])])
  cache, values = S.cache(rng, 2 * kv, int(first[-1]) + 3, hd, fmt)
  qb = torch.from_numpy(rng.normal(0, 0.1, (sum(lens), heads * hd)).astype(np.float32)).to(S.DTYPE[q])
  starts = np.concatenate([[0], np.cumsum(lens)])
  got = ops().attention_prefill_packed(qb.cuda(), cache, heads, kv, hd, ints(starts), ints(cached), ints(first[:-1]), max(a + c for a, c in zip(lens, cached)),
                                       out_dtype=torch.bfloat16)
  for s, (a, c) in enumerate(zip(lens, cached)):
    lo = int(starts[s])
    want, tol = attend(qb[lo:lo + a], values, torch.arange(a + c) + int(first[s]), c + 1 + np.arange(a), kv, hd)
    check(got[lo:lo + a], want, tol, s)


@pytest.mark.parametrize("heads,kv,hd,fmt,q", HEADS)
@pytest.mark.parametrize("batch,prefix,own", [(3, 20, 5), (17, 300, 90), (4, 2000, 700)])
@pytest.mark.parametrize("tiles", [False, True])
def test_shared_bf16_output(cuda, heads, kv, hd, fmt, q, batch, prefix, own, tiles):
  # (what attention_decode keeps its weights to, so that a step behind a shared prefix loses nothing)
  print(f"shared bf16 {batch} {prefix} {own} {heads}/{kv} {hd} {fmt} {q} {tiles}", flush=True)
  rng = np.random.default_rng(72)
  mine = rng.integers(1, own + 1, batch)
  first = prefix + 4 + np.concatenate([[0], np.cumsum(mine)])
  cache, values = S.cache(rng, 2 * kv, int(first[-1]) + 3, hd, fmt)
  qb = torch.from_numpy(rng.normal(0, 0.1, (batch, heads * hd)).astype(np.float32)).to(S.DTYPE[q])
  got = ops().attention_decode_shared(qb.cuda(), cache, heads, kv, hd, ints(prefix + mine - 1), ints(first[:-1]), ints([2]), ints([prefix] * batch), prefix, own,
                                      o=ops().tiles16(batch, heads * hd) if tiles else None, out_dtype=torch.bfloat16)
  if tiles: got = got.to_rows()
  for b in range(batch):
    where = S.rows_of(2, prefix, int(first[b]), prefix + int(mine[b]))
    want, tol = attend(qb[b:b + 1], values, where, [len(where)], kv, hd)
    check(got[b:b + 1], want, tol, b)


def test_rows_given_on_the_gpu_behind_the_places_their_slots_were_filled_behind(cuda):
  # places and slots as tensors on the GPU: the same cache rows, steps and refusals as the host's
  from test_gpu_20_serving import decoder
  rng = np.random.default_rng(73)
  prompt = lambda n: [int(i) for i in rng.integers(0, 2048, n)]
  dec = decoder(74, "bf16", 3, 100, 4)
  dec.prefill(prompt(70), slot=3)
  dec.share_prefix(3, 70, rows=[70, 35, 0])
  prompts = [prompt(n) for n in (5, 9, 20)]
  dec.prefill_batch(prompts)
  with pytest.raises(ValueError, match="slot 1 holds"): dec.step([1, 2, 3], ints([75, 44, 20]), ints([0, 1, 2]))
  dec.prefill_batch(prompts, shared=[70, 35, 0])
  got = dec.step([1, 2, 3], ints([75, 44, 20]), ints([0, 1, 2]))[0].clone()
  assert torch.equal(got, dec.step([1, 2, 3], [75, 44, 20], [0, 1, 2])[0]) and dec.rows.tolist() == [5, 109, 220]


def test_one_workspace_for_a_services_largest_calls(cuda):
  # taken once for the largest batch and bounds, it serves smaller ones, whose keys are split where the largest's are not
  rng = np.random.default_rng(75)
  heads, kv, hd = 32, 8, 128
  cache, values = S.cache(rng, 2 * kv, 5000, hd, "bf16")
  ws = ops().attention_packed_workspace(8192, 16, heads, kv, hd, 4096)
  ws.fill_(255)
  for lens, cached in (([200], [3000]), ([3], [4090]), ([40, 30], [500, 9])):
    first = np.concatenate([[0], np.cumsum([a + c for a, c in zip(lens, cached)])])
    starts = np.concatenate([[0], np.cumsum(lens)])
    q = torch.from_numpy(rng.normal(0, 0.1, (sum(lens), heads * hd)).astype(np.float32))
    got = ops().attention_prefill_packed(q.cuda(), cache, heads, kv, hd, ints(starts), ints(cached), ints(first[:-1]), 4096, workspace=ws, out_dtype=torch.bfloat16)
    for s, (a, c) in enumerate(zip(lens, cached)):
      lo, some = int(starts[s]), slice(max(0, a - 7), a)  # (the last rows of each, in 64 bits)
      want, tol = attend(q[lo:lo + a][some], values, torch.arange(a + c) + int(first[s]), (c + 1 + np.arange(a))[some], kv, hd)
      check(got[lo:lo + a][some], want, tol, (lens, s))
  ws = ops().attention_shared_workspace(16, heads, kv, hd, 4096, 4096)
  ws.fill_(255)
  for batch, prefix, own in ((16, 4096, 40), (3, 4000, 300), (1, 10, 900)):
    first = prefix + np.arange(batch) * 50
    mine = rng.integers(1, own + 1, batch)
    q = torch.from_numpy(rng.normal(0, 0.1, (batch, heads * hd)).astype(np.float32))
    got = ops().attention_decode_shared(q.cuda(), cache, heads, kv, hd, ints(prefix + mine - 1), ints(first), ints([0]), ints([prefix] * batch), prefix, own,
                                        workspace=ws, out_dtype=torch.bfloat16)
    for b in range(batch):
      where = S.rows_of(0, prefix, int(first[b]), prefix + int(mine[b]))
      want, tol = attend(q[b:b + 1], values, where, [len(where)], kv, hd)
      check(got[b:b + 1], want, tol, (batch, b))


def test_the_captured_step_after_other_counts_and_another_slot(cuda):
  # the same graph, replayed after share_prefix gave other counts and another slot of the same length, against eager steps
  from test_gpu_20_serving import decoder
  rng = np.random.default_rng(76)
  prompt = lambda n: [int(i) for i in rng.integers(0, 2048, n)]
  dec = decoder(77, "bf16", 3, 100, 5)
  for slot in (3, 4): dec.prefill(prompt(70), slot=slot)
  prompts, graph = [prompt(n) for n in (5, 9, 20)], None
  for slot, counts in ((3, [70, 70, 70]), (3, [70, 35, 0]), (4, [70, 35, 0]), (4, [0, 70, 12])):
    dec.share_prefix(slot, 70, rows=counts)
    dec.prefill_batch(prompts, shared=counts)
    places = [n + len(p) for n, p in zip(counts, prompts)]
    want = dec.step([1, 2, 3], places, [0, 1, 2], replay=False)[0].clone()
    for _ in range(2): assert torch.equal(dec.step([1, 2, 3], places, [0, 1, 2])[0], want), (slot, counts)
    assert graph is None or dec.graph is graph
    graph = dec.graph


@pytest.mark.parametrize("batch,prefix,own,bound", [(16, 200, 2500, 4096), (2, 65, 4000, 8192), (16, 300, 90, 1 << 30)])
def test_many_own_keys_behind_a_short_prefix(cuda, batch, prefix, own, bound):
  # the rows' own keys split over most of the GPU; a bound far above what is there
  print(f"own keys {batch} {prefix} {own} {bound}", flush=True)
  rng = np.random.default_rng(78)
  heads, kv, hd = 32, 8, 128
  mine = rng.integers(1, own + 1, batch)
  mine[0] = own
  first = prefix + 4 + np.concatenate([[0], np.cumsum(mine)])
  cache, values = S.cache(rng, 2 * kv, int(first[-1]) + 3, hd, "bf16")
  q = torch.from_numpy(rng.normal(0, 0.1, (batch, heads * hd)).astype(np.float32))
  got = ops().attention_decode_shared(q.cuda(), cache, heads, kv, hd, ints(prefix + mine - 1), ints(first[:-1]), ints([2]), ints([prefix] * batch), prefix, bound,
                                      out_dtype=torch.bfloat16)
  for b in range(batch):
    where = S.rows_of(2, prefix, int(first[b]), prefix + int(mine[b]))
    want, tol = attend(q[b:b + 1], values, where, [len(where)], kv, hd)
    check(got[b:b + 1], want, tol, b)
