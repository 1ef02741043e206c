"""The cache in pages and the adapters where their other tests do not go; each test says what it holds to."""
import numpy as np
import pytest
import torch
import seq_cases as S
from test_gpu_23_paged import ints, ops
from test_gpu_26_pages import LAYERS, VOCAB, adapters_of, close, config, decoder, pages_for
from oracle import llama as OL

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["fp32", "bf16", "bfp8", "bfp4"])
@pytest.mark.parametrize("hd,x,T", [(64, "fp32", 5), (128, "bf16", 5), (128, "fp32", 1100)])
def test_a_heads_norm_whose_squares_overflow(cuda, fmt, hd, x, T):
  # A head of values past 2^64: the mean of their squares is infinite in 32 bits and the norm 0, as the framework's other norms give;
  # a block float's keys, normed in 64 bits, are the formula's (values alike: 1). The other heads and rows keep their bits.
  print(f"huge {fmt} {hd} {x} {T}", flush=True)
  rng = np.random.default_rng(91)
  heads, kv, pages = 3, 2, -(-T // 16)
  rows = torch.from_numpy(rng.normal(0, 1, (T, heads + 2 * kv, hd)).astype(np.float32)).to(S.DTYPE[x]).cuda()
  huge = rows.clone()
  huge[2 % T, 1], huge[2 % T, heads] = 2.0 ** 65, -2.0 ** 66
  w, out = torch.ones(hd, device="cuda"), []
  for v in (rows, huge):
    cache = ops().kv_cache(2 * kv, 16 * pages, hd, fmt)
    (cache.data if fmt in ("bfp8", "bfp4") else cache).zero_()
    q = ops().rope_append_paged(v.view(T, -1), cache, heads, kv, hd, None, None, ints([0, T]), ints([0]), ints(range(pages)).view(1, -1), 16, q_norm=w, k_norm=w, eps=1e-5)
    if fmt in ("bfp8", "bfp4"):
      n = 2 * kv * 16 * pages
      wide = hd if fmt == "bfp8" else hd // 2
      held = (cache.data[:n * wide].view(2 * kv, -1, wide).clone(), cache.data[n * wide:].view(2 * kv, -1, hd // 16).clone())
    else: held = (cache.clone(),)
    out.append((q.view(T, heads, hd), held))
  (q0, c0), (q1, c1) = out
  at = 2 % T
  assert (q1[at, 1] == 0).all() and torch.isfinite(q1).all()
  # values whose squares vanish, with no eps: a mean of 2^-140, below the normal numbers, and 1
  tiny = torch.full((1, (heads + 2 * kv) * hd), 2.0 ** -70, device="cuda").to(S.DTYPE[x])
  q = ops().rope_append_paged(tiny, ops().kv_cache(2 * kv, 16, hd, fmt), heads, kv, hd, None, None, ints([0, 1]), ints([0]), ints([0]).view(1, 1), 16, q_norm=w, k_norm=w, eps=0.0)
  assert float((q - 1).abs().max()) <= 24 * 2.0 ** -24
  keep = torch.ones(T, heads, dtype=torch.bool, device="cuda")
  keep[at, 1] = False
  assert torch.equal(q0[keep], q1[keep])
  for a, b in zip(c0, c1):
    keep = torch.ones(a.shape[:2], dtype=torch.bool, device="cuda")
    keep[0, at] = False
    assert torch.equal(a[keep], b[keep])
  if fmt in S.DTYPE: assert (c1[0][0, at] == 0).all()
  else:  # -1: whole steps of 2^-6 or 2^-2 under the exponent of 1, two to a byte in bfp4
    m = c1[0][0, at]
    assert (c1[1][0, at] == 127).all() and (m == (256 - 64 if fmt == "bfp8" else 0xCC)).all()


def far(seed, heads, kv, hd, lens, before, bound, fmt="bf16", q="fp32", o="bf16", page=1 << 12, cols=1 << 18):
  """A call whose max_context is `bound`, over few pages that many sequences read, against the formula."""
  rng = np.random.default_rng(seed)
  n, some = len(lens), 3
  cache, values = S.cache(rng, 2 * kv, some * page, hd, fmt)
  pick = rng.integers(0, some, n)
  tables = torch.full((n, cols), -5, dtype=torch.int32, device="cuda")
  tables[:, 0] = ints(pick)
  starts = np.concatenate([[0], np.cumsum(lens)])
  qb = torch.from_numpy(rng.normal(0, 1.5, (int(starts[-1]), heads * hd)).astype(np.float32)).to(S.DTYPE[q])
  assert max(a + b for a, b in zip(lens, before)) <= page and bound <= cols * page
  got = ops().attention_paged(qb.cuda(), cache, heads, kv, hd, ints(starts), ints(before), tables, page, bound, out_dtype=S.DTYPE[o])
  want, tol = torch.zeros(got.shape, dtype=torch.float64), torch.zeros(got.shape, dtype=torch.float64)
  for s in range(n):
    a, b, lo = lens[s], before[s], int(starts[s])
    if a: want[lo:lo + a], tol[lo:lo + a] = S.attend(qb[lo:lo + a], values, pick[s] * page + torch.arange(a + b), b + 1 + np.arange(a), kv, hd, o == "bf16")
  S.check(got, want, tol, (lens, bound, fmt))


@pytest.mark.parametrize("bits", [24, 26, 28, 30])
@pytest.mark.parametrize("heads,kv,hd,fmt,q,o", [(4, 2, 64, "bf16", "fp32", "bf16"), (4, 1, 128, "bfp8", "bf16", "fp32"), (2, 1, 64, "fp32", "fp32", "fp32"),
                                                 (8, 1, 128, "bf16", "bf16", "bf16")])
def test_costs_in_units(cuda, bits, heads, kv, hd, fmt, q, o):
  # bounds so large that a call's costs go in units of 2 to 2^11 keys (tiles times max_context from 2^30 on): prompts of several tiles, chunks
  # after many places, tokens beside them and single tokens alone
  print(f"units {bits} {heads}/{kv} {hd} {fmt} {q} {o}", flush=True)
  far(92, heads, kv, hd, [150, 1, 0, 129, 20, 1, 70], [0, 3000, 7, 1500, 2, 0, 3800], 1 << bits, fmt, q, o)
  far(93, heads, kv, hd, [1] * 70, [int(b) for b in np.random.default_rng(1).integers(0, 2500, 70)], 1 << bits, fmt, q, o)
  if bits == 30: far(94, heads, kv, hd, [1] * 900, [int(b) for b in np.random.default_rng(2).integers(0, 60, 900)], 1 << bits, fmt, q, o)


@pytest.mark.parametrize("fmt,q,o", [("bfp8", "fp32", "bf16"), ("bfp4", "bf16", "bf16"), ("bfp8", "bf16", "fp32"), ("fp32", "fp32", "fp32")])
def test_block_floats_and_fp32_repeat_their_bits(cuda, fmt, q, o):
  # prompts, chunks and tokens cut over many workgroups: every call gives the same bits, on two streams at a time as well
  rng = np.random.default_rng(95)
  heads, kv, hd, n = 20, 4, 64, 11
  cache, _ = S.cache(rng, 2 * kv, 32 * 300, hd, fmt)
  lens = [250, 1, 130, 77, 0, 199, 1, 64, 128, 1, 90]
  starts = ints(np.concatenate([[0], np.cumsum(lens)]))
  x = torch.from_numpy(rng.normal(0, 1.5, (sum(lens), heads * hd)).astype(np.float32)).to(S.DTYPE[q]).cuda()
  tables = torch.from_numpy(rng.integers(0, 300, (n, 40)).astype(np.int32)).cuda()
  args = (x, cache, heads, kv, hd, starts, ints(rng.integers(0, 900, n)), tables, 32, 1200)
  want = ops().attention_paged(*args, out_dtype=S.DTYPE[o])
  torch.cuda.synchronize()
  streams, outs = [torch.cuda.Stream() for _ in range(2)], []
  for i in range(24):
    with torch.cuda.stream(streams[i % 2]): outs.append(ops().attention_paged(*args, out_dtype=S.DTYPE[o]))
  torch.cuda.synchronize()
  assert all(torch.equal(t, want) for t in outs)


def mantissas(rng, *shape):
  """fp32 values of 24 random bits each, 1 to 2 and their negatives."""
  return torch.from_numpy(((rng.integers(1 << 23, 1 << 24, shape) | 1) * 2.0 ** -23 * rng.choice([-1.0, 1.0], shape)).astype(np.float32))


@pytest.mark.parametrize("T,K,N,rank", [(9, 64, 96, 16), (70, 576, 192, 8), (130, 328, 264, 40), (33, 1000, 64, 128)])
@pytest.mark.parametrize("x", ["fp32", "bf16"])
@pytest.mark.parametrize("w", ["fp32", "bf16"])
def test_fp32_adapters_to_their_last_term(cuda, T, K, N, rank, x, w):
  # One value in each row of x, one in each column of A's product that meets it, one in each row of B: nothing is added but a product's own
  # terms, so that what is left of the error is theirs. A value of 24 bits is its three terms' sum exactly (8 bits each, signed), and a product by a
  # power of two is exact. Of two values of 24 bits a product's terms i + j > 2 are left out: twice 2^-8 2^-16 and 2^-32 of it; the 6 kept
  # are added in 32 bits, at most 6 half steps (2^-24 of sums up to 1 + 2^-7 of it; twice that if the matrix core truncates). u and y
  # are each such a product: (2 + 2 * 6) 2^-24 of it at u, the same at y and u's rounding to 24 bits.
  print(f"lora terms {T} {K} {N} {rank} {x} {w}", flush=True)
  rng = np.random.default_rng(96)
  bf = lambda t, kind: t if kind == "fp32" else t.to(torch.bfloat16).float()
  for full in ("x", "a", "b", "all"):
    two = lambda *s: torch.from_numpy((2.0 ** rng.integers(-3, 4, s) * rng.choice([-1.0, 1.0], s)).astype(np.float32))
    make = lambda name, *s: mantissas(rng, *s) if full in (name, "all") else two(*s)
    k_of, r_of = rng.integers(0, K, T), rng.integers(0, rank, N)
    xs = torch.zeros(T, K)
    xs[torch.arange(T), torch.from_numpy(k_of)] = bf(make("x", T), x)
    a, b = bf(make("a", 1, rank, K), w), torch.zeros(1, N, rank)
    b[0, torch.arange(N), torch.from_numpy(r_of)] = bf(make("b", N), w)
    ad = ops().Adapters(a.to(S.DTYPE[w]).cuda(), b.to(S.DTYPE[w]).cuda(), None, (N,))
    got = ops().lora(xs.to(S.DTYPE[x]).cuda(), ad, ints([0] * T)).double().cpu()
    want = (xs.double() @ a[0].double().T) @ b[0].double().T
    tol = 0 if full != "all" else 30 * 2.0 ** -24
    err = (got - want).abs() / want.abs().clamp(min=2.0 ** -100)
    assert (want != 0).all() and float(err.max()) <= tol, (full, float(err.max()) * 2 ** 24)


@pytest.mark.parametrize("fmt", ["bf16", "bfp8", "bfp4", "fp32"])
@pytest.mark.parametrize("hd,heads,kv", [(64, 4, 2), (128, 4, 1)])
@pytest.mark.parametrize("tokens", [False, True])
def test_fp32_attention_to_its_last_term(cuda, fmt, hd, heads, kv, tokens):
  # One value in each row of q (24 bits) and of v, powers of 2 in k and v: a score is one product, its terms' sum exact, and each output one weight
  # times a power of 2. What is left: the scale, two roundings and the constant's (2.5 half steps of |s|), the exponent's fma (one of at most 2 |s|) and its
  # exp2 (2), once for the weight and once for the sum, whose n additions are a half step each, and 4 for the quotient and the
  # output: (9 |s| + 8 + n) 2^-24. A third term left out of q moves a weight by up to 5e-5 where scores are 4 to 8 (allowed: 7e-6), out of a
  # weight the output by up to 5e-6 (allowed: 3e-6 where scores are small).
  print(f"attention terms {fmt} {hd} {heads}/{kv} {tokens}", flush=True)
  rng, n = np.random.default_rng(100), 40
  t = torch.arange(n)
  for base, most in ((hd ** 0.5 * 4, 8.0), (hd ** 0.5 / 8, 0.25)):
    base = 2.0 ** round(np.log2(base))
    most *= base / (hd ** 0.5 * 4 if most == 8.0 else hd ** 0.5 / 8)
    sign = lambda *s: torch.from_numpy(rng.choice([-1.0, 1.0], s).astype(np.float32))
    q, k, v = torch.zeros(n, heads, hd), sign(n, kv, hd) * base * torch.from_numpy((2.0 ** -rng.integers(0, 3, (n, kv, hd))).astype(np.float32)), torch.zeros(n, kv, hd)
    for h in range(heads): q[t, h, torch.from_numpy(rng.integers(0, hd, n))] = mantissas(rng, n)
    for h in range(kv): v[t, h, t] = sign(n) * torch.from_numpy((2.0 ** rng.integers(-2, 3, n)).astype(np.float32))
    cache = ops().kv_cache(2 * kv, 64, hd, fmt)
    table, x = [[2, 0, 3]], torch.cat([q, k, v], 1).reshape(n, -1).cuda()
    qx = ops().rope_append_paged(x, cache, heads, kv, hd, None, None, ints([0, n]), ints([0]), torch.tensor(table, dtype=torch.int32, device="cuda"), 16)
    args = (ints(range(n + 1)), ints(range(n)), torch.tensor(table * n, dtype=torch.int32, device="cuda")) if tokens else (ints([0, n]), ints([0]), torch.tensor(table, dtype=torch.int32, device="cuda"))
    got = ops().attention_paged(qx, cache, heads, kv, hd, *args, 16, n).double().cpu().view(n, heads, hd)
    for h in range(heads):
      g = h // (heads // kv)
      s = (q[:, h].double() @ k[:, g].double().T) / np.sqrt(hd)
      p = torch.softmax(s.masked_fill(t[None] > t[:, None], -np.inf), 1)
      want = p @ v[:, g].double()
      assert float(s.abs().max()) <= most
      off = ((got[:, h] - want).abs() / want.abs().clamp(min=1e-30))[want != 0]
      assert float(off.max()) <= (9 * most + 8 + n) * 2.0 ** -24 and (got[:, h][want == 0] == 0).all(), (h, base, float(off.max()) * 2 ** 24)


def test_a_model_of_grouped_heads_of_128_dimensions(cuda):
  # prompts, chunks and tokens in pages, then replayed steps, against its slots
  from ferrite_amd import llama as G
  cfg = dict(dim=512, heads=8, kv=2, head_dim=128, layers=2, eps=1e-5, theta=10000.0, vocab=1024, ffn=768, places=400)
  for kv, page in (("bf16", 32), ("bfp8", 16)):
    rng = np.random.default_rng(97)
    slots = G.Decoder(G.model(**cfg), G.numpy_weights(OL.random_weights(OL.model(**cfg), rng)), mode="bfp8", kv=kv, batch=1, context=320, slots=3)
    dec = G.Decoder(G.model(**cfg), None, mode="bfp8", kv=kv, batch=1, context=320, slots=3, share=slots)
    text = [[int(i) for i in rng.integers(0, 1024, 300)] for _ in range(3)]
    tables = pages_for(rng, [-(-300 // page)] * 3, 960 // page)
    at = [0] * 3
    def want(i, n): return slots.prefill(text[i][at[i]:at[i] + n], slot=i, p0=at[i])[0].clone()
    for lens in ([170, 1, 33], [1, 90, 40], [20, 1, 1]):
      got = dec.step_pages([text[i][at[i]:at[i] + n] for i, n in enumerate(lens)], at, tables, page)[0]
      close(got, torch.cat([want(i, n) for i, n in enumerate(lens)]), (kv, lens))
      at = [a + n for a, n in zip(at, lens)]
    step = dec.page_step(3, -(-300 // page), page)
    for _ in range(3):
      got = step.step([text[i][at[i]] for i in range(3)], at, tables)[0]
      close(got, torch.cat([want(i, 1) for i in range(3)]), (kv, "step"))
      at = [a + 1 for a in at]


def test_a_decode_step_takes_its_own_picks(cuda):
  # the picks of step_pages and of each step, int32 on the GPU, are the next step's tokens as they are
  rng = np.random.default_rng(98)
  dec = decoder(OL.random_weights(config()[0], rng), "bf16", 160, 3)
  text = [[int(i) for i in rng.integers(0, VOCAB, n)] for n in (30, 7, 1)]
  tables, places = pages_for(rng, [5] * 3, 30), [30, 7, 1]
  picks = dec.step_pages(text, [0, 0, 0], tables, 16)[1]
  step = dec.page_step(3, 5, 16)
  for i in range(4):
    tokens = picks.tolist()
    logits, now = step.step(picks, places, tables)
    got = (logits.clone(), now.clone())
    want = step.step(tokens, places, tables)   # (the same tokens at the same places, from the host)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    also = step.step(got[1].new_tensor(tokens).long(), places, tables, replay=False)
    assert torch.equal(also[0], got[0])
    picks, places = want[1], [p + 1 for p in places]
  for bad in (picks[:2], picks.view(3, 1), picks.float()):
    with pytest.raises(ValueError, match="tokens"): step.step(bad, places, tables)


def test_a_step_keeps_the_adapters_it_was_made_with(cuda):
  # the caller puts others into its own lists after the step was made and captured, and their memory is given to something else
  rng = np.random.default_rng(99)
  dec = decoder(OL.random_weights(config()[0], rng), "bf16", 160, 2)
  ads = adapters_of(rng, 2, ("qkv", "down"), 8)[0]
  sizes = [(a.a.shape, a.b.shape) for ad in ads for a in ad.values()]
  call = lambda s, **kw: s.step([5, 9], [0, 3], [[0, 1], [2, 3]], [1, 0], **kw)[0].clone()
  step = dec.page_step(2, 2, 16, ads)
  want = call(step)
  other = adapters_of(rng, 2, ("qkv", "down", "gate_up"), 24)[0]
  for l in range(LAYERS):
    ads[l]["qkv"], ads[l]["down"], ads[l]["gate_up"] = other[l]["qkv"], other[l]["down"], other[l]["gate_up"]
  ads.append({})
  torch.cuda.synchronize()
  junk = [torch.full(s, float("nan"), dtype=torch.bfloat16, device="cuda") for pair in sizes for s in pair for _ in range(4)]
  torch.cuda.synchronize()
  assert torch.equal(call(step), want) and torch.equal(call(step, replay=False), want) and len(junk)
  assert not torch.equal(call(dec.page_step(2, 2, 16, ads[:LAYERS])), want)
