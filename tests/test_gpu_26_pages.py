"""The model over a cache in pages (Decoder.step_pages, page_step) with and without low-rank adapters: against the Decoder's slots (prefill,
tested against numpy) and against numpy with each adapter's products, within the bar the logits are held to there (1e-2 of the
largest, cosine 0.9999)."""
import numpy as np
import pytest
import torch
from oracle import llama as OL

pytestmark = pytest.mark.gpu
LAYERS, VOCAB = 2, 2048


def config():
  from ferrite_amd import llama as G
  c = OL.smollm(layers=LAYERS, vocab=VOCAB, places=400)
  return c, G.model(**{k: getattr(c, k) for k in ("dim", "heads", "kv", "layers", "eps", "theta", "vocab", "ffn", "places", "rope", "tied")})


def decoder(w, kv, context, slots, share=None):
  from ferrite_amd import llama as G
  return G.Decoder(config()[1], None if share is not None else G.numpy_weights(w), mode="bfp8", kv=kv, batch=1, context=context, slots=slots, share=share)


def close(got, want, what):
  got, want = torch.as_tensor(got).double().cpu(), torch.as_tensor(want).double().cpu()
  rel = float((got - want).abs().max() / want.abs().max())
  cos = float((got * want).sum() / (got.norm() * want.norm()))
  assert rel <= 1e-2 and cos >= 0.9999, (what, rel, cos)


def adapters_of(rng, n, names, rank):
  """For each block the named projections' adapters, and the matrices they are made of."""
  from ferrite_amd import ops
  c, _ = config()
  hd = c.dim // c.heads
  shapes = dict(qkv=(c.dim, (c.heads * hd, c.kv * hd, c.kv * hd)), o=(c.heads * hd, (c.dim,)), gate_up=(c.dim, (c.ffn, c.ffn)), down=(c.ffn, (c.dim,)))
  blocks, mats = [], []
  bf = lambda a: torch.from_numpy(a.astype(np.float32)).to(torch.bfloat16)
  for _ in range(LAYERS):
    ad, m = {}, {}
    for name in names:
      K, parts = shapes[name]
      m[name] = [[(bf(rng.normal(0, 2 * K ** -0.5, (rank, K))), bf(rng.normal(0, 0.3, (p, rank)))) for p in parts] for _ in range(n)]
      ad[name] = ops.pack_adapters(m[name], parts, scales=[1.0 + 0.5 * i for i in range(n)])
    blocks.append(ad)
    mats.append(m)
  return blocks, mats


def forward64(tokens, arrays, c, adapters, rounded=True):
  """The model in 64 bits for one sequence, every row's logits; rounded: with the Decoder's own roundings, each product's rows in bf16."""
  bf = (lambda a: torch.from_numpy(a.astype(np.float32)).to(torch.bfloat16).double().numpy()) if rounded else (lambda a: a)
  T, hd, rep = len(tokens), c.dim // c.heads, c.heads // c.kv
  def rms(x, w): return bf(x / np.sqrt((x * x).mean(1, keepdims=True) + c.eps) * w)
  def product(l, name, full, x):
    y = x @ arrays[f"layers.{l}.{full}"].astype(np.float64)
    scale, parts = adapters(l, name)
    return y if parts is None else y + scale * np.concatenate([(x @ A.double().numpy().T) @ B.double().numpy().T for A, B in parts], 1)
  x = arrays["embed"][list(tokens)].astype(np.float64)
  cos, sin = (t[:T, None, :hd].astype(np.float64) for t in OL.rotary_head(c, T))
  for l in range(LAYERS):
    qkv = product(l, "qkv", "qkv_proj", rms(x, arrays[f"layers.{l}.input_layernorm"])).reshape(T, -1, hd)
    qk, v = qkv[:, :c.heads + c.kv], qkv[:, c.heads + c.kv:]
    qk = qk * cos + np.concatenate([-qk[..., hd // 2:], qk[..., :hd // 2]], -1) * sin
    out = np.zeros((T, c.heads, hd))
    for h in range(c.heads):
      s = np.where(np.tri(T, dtype=bool), qk[:, h] @ qk[:, c.heads + h // rep].T / np.sqrt(hd), -np.inf)
      e = np.exp(s - s.max(1, keepdims=True))
      out[:, h] = e / e.sum(1, keepdims=True) @ v[:, h // rep]
    x = x + product(l, "o", "o_proj", bf(out.reshape(T, -1)))
    gu = product(l, "gate_up", "gate_up_proj", rms(x, arrays[f"layers.{l}.post_attention_layernorm"]))
    g, u = gu[:, :c.ffn], gu[:, c.ffn:]
    x = x + product(l, "down", "down_proj", bf(g / (1 + np.exp(-g)) * u))
  return rms(x, arrays["norm"]) @ arrays["embed.T"].astype(np.float64)


def pages_for(rng, counts, total):
  ids, at, out = rng.permutation(total), 0, []
  for n in counts:
    out.append([int(i) for i in ids[at:at + n]])
    at += n
  return out


@pytest.mark.parametrize("kv,page", [("bf16", 16), ("fp32", 64), ("bfp8", 32)])
def test_pages_as_slots(cuda, kv, page):
  # prompts, a second turn in chunks beside single tokens, then replayed decode steps: each sequence's logits as its own slot gives them
  rng = np.random.default_rng(71)
  w = OL.random_weights(config()[0], rng)
  slots = decoder(w, kv, 320, 4)
  dec = decoder(w, kv, 320, 4, share=slots)
  text = [[int(i) for i in rng.integers(0, VOCAB, 300)] for _ in range(4)]
  tables = pages_for(rng, [-(-300 // page)] * 4, 1280 // page)
  at = [0] * 4
  def go(lens, which):
    got, picks = dec.step_pages([text[i][at[i]:at[i] + n] for i, n in zip(which, lens)], [at[i] for i in which], [tables[i] for i in which], page)
    want = torch.cat([slots.prefill(text[i][at[i]:at[i] + n], slot=i, p0=at[i])[0].clone() for i, n in zip(which, lens)])
    close(got, want, (lens, which))
    assert torch.equal(picks.long().cpu(), got.argmax(1).cpu())
    for i, n in zip(which, lens): at[i] += n
  go([40, 1, 130, 65], [0, 1, 2, 3])
  go([1, 90, 1], [0, 1, 3])
  go([1], [2])
  step = dec.page_step(3, -(-300 // page), page)
  for which in ([3, 0, 2], [0, 1, 2], [2, 3, 1]):
    got, picks = step.step([text[i][at[i]] for i in which], [at[i] for i in which], [tables[i] for i in which])
    want = torch.cat([slots.prefill([text[i][at[i]]], slot=i, p0=at[i])[0].clone() for i in which])
    close(got, want, ("replay", which))
    assert torch.equal(picks.long().cpu(), got.argmax(1).cpu())
    again = step.step(replay=False)[0]
    assert torch.equal(again, got)
    for i in which: at[i] += 1
    go([2, 3], which[:2])  # (the program's own work between replays)


def test_a_common_prompt_in_common_pages(cuda):
  # two sequences whose tables begin with the same pages, filled once
  rng = np.random.default_rng(72)
  dec = decoder(OL.random_weights(config()[0], rng), "bf16", 320, 2)
  system, a, b = ([int(i) for i in rng.integers(0, VOCAB, n)] for n in (64, 20, 7))
  common = [5, 9, 2, 11]
  dec.step_pages([system], [0], [common], 16)
  got = dec.step_pages([a, b], [64, 64], [common + [7, 8], common + [3]], 16)[0]
  for i, t in enumerate((a, b)):
    close(got[i:i + 1], dec.step_pages([system + t], [0], [list(range(20, 26))], 16)[0], i)
  with pytest.raises(ValueError, match="another's"): dec.step_pages([a, b], [60, 64], [common + [7, 8], common + [3]], 16)


@pytest.mark.parametrize("names", [("qkv",), ("o", "down"), ("gate_up",), ("qkv", "o", "gate_up", "down")])
def test_adapters(cuda, names):
  rng = np.random.default_rng(73)
  c, _ = config()
  w = OL.random_weights(c, rng)
  dec = decoder(w, "fp32", 160, 4)
  blocks, mats = adapters_of(rng, 3, names, 12)
  lens, of = [30, 1, 55, 9], [2, 0, -1, 1]
  text = [[int(i) for i in rng.integers(0, VOCAB, n + 1)] for n in lens]
  tables = pages_for(rng, [5] * 4, 40)
  got = dec.step_pages([t[:-1] for t in text], [0] * 4, tables, 16, blocks, of)[0]
  step = dec.page_step(4, 5, 16, blocks)
  nxt = step.step([t[-1] for t in text], lens, tables, of)[0]
  plain = dec.step_pages([text[0][:-1]], [0], [tables[0]], 16)[0]
  c.precision = OL.precision(c, "bfp8", "fp32")
  arrays = OL.arrays(w, c.precision)
  for i, t in enumerate(text):
    given = lambda l, name: (1.0 + 0.5 * of[i], mats[l][name][of[i]]) if of[i] >= 0 and name in names else (0, None)
    want, exact = forward64(t, arrays, c, given), forward64(t, arrays, c, given, False)
    # Strong adapters sharpen the attention, and with it every rounding of a row. The GPU takes the oracle's roundings, but its rows come from
    # sums of K products in 32 bits, off by about sqrt(K) 2^-24 of a few times themselves, so of the values, whose bf16 steps are 2^-8 to
    # 2^-7 of them, about 2 * 4 sqrt(1536) 2^-24 / 2^-8, one in 200, is rounded to the other side, off by a step where all the others' roundings are off
    # by 0.29 of one in the mean: together sqrt(1 / 200) / 0.29, a quarter, of what the roundings move the logits by, which is the bound
    for g, w64, e64 in ((got[i], want[-2], exact[-2]), (nxt[i], want[-1], exact[-1])):
      off = float(np.linalg.norm(g.double().cpu().numpy() - w64))
      assert off <= max(float(np.linalg.norm(w64 - e64)), 1e-3 * float(np.linalg.norm(w64))), (i, off, float(np.linalg.norm(w64 - e64)), float(np.linalg.norm(w64)))
      if of[i] < 0 or len(names) == 1: close(g, w64, i)
  assert float((plain[0] - got[0]).abs().max()) > 0.05 * float(got[0].abs().max())  # (the adapters are not nothing)


def test_step_pages_refuses(cuda):
  from ferrite_amd import ops
  rng = np.random.default_rng(74)
  dec = decoder(OL.random_weights(config()[0], rng), "bf16", 160, 2)
  ok = dict(tokens=[[1, 2], [3]], places=[0, 5], tables=[[0], [1]], page=16)
  dec.step_pages(**ok)
  for kw in (dict(tokens=[]), dict(tokens=[[], [1]]), dict(places=[0]), dict(places=[-1, 0]), dict(places=[0, 400]), dict(places=[15, 0]), dict(tables=[[0]]), dict(tables=[[0], []]),
             dict(tables=[[0], [20]]), dict(tables=[[0], [-1]]), dict(tables=[[1], [1]]), dict(page=8), dict(page=24), dict(page=128), dict(of=[0]), dict(adapters=[{}, {}, {"o": None}])):
    with pytest.raises(ValueError): dec.step_pages(**(ok | kw))
  wrong = ops.Adapters(torch.zeros(1, 8, 576, device="cuda"), torch.zeros(1, 64, 8, device="cuda"), None, (64,))
  for kw in (dict(adapters=[{"o": wrong}, {}]), dict(adapters=[{"x": wrong}, {}])):
    with pytest.raises(ValueError): dec.step_pages(**(ok | kw))
    with pytest.raises(ValueError): dec.page_step(2, 4, 16, **kw)
  for kw in (dict(n=0), dict(pages=0), dict(page=48)):
    with pytest.raises(ValueError): dec.page_step(**(dict(n=2, pages=4, page=16) | kw))
  s = dec.page_step(2, 2, 16)
  with pytest.raises(ValueError): s.step([1, 2], [0, 0], [[0], [0]])
  with pytest.raises(ValueError): s.step([1, 2], [40, 0], [[0, 1, 2], [3]])
  with pytest.raises(ValueError): s.step([1], [0, 0], [[0], [1]])
