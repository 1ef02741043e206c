"""A batch served from end to end: a system prompt prefilled once and shared, the requests' prompts packed together behind
it, greedy steps replayed as one graph, and each step's heads under the requests' rules; against a Decoder that holds every
sequence whole in its own slot, prefilled one at a time (the path tested against numpy), within the bar its logits are held to
there (1e-2 of the largest, cosine 0.9999), and the heads against numpy on the step's own logits."""
import numpy as np
import pytest
import torch
from oracle import llama as OL
from oracle.serve import head_of

pytestmark = pytest.mark.gpu
SYSTEM, PROMPTS = 70, [5, 33, 1, 64, 18]


def decoder(seed, kv, batch, context, slots, share=None, mfma_from=3, layers=2):
  from ferrite_amd import llama as G
  c = OL.smollm(layers=layers, vocab=2048, places=400)
  gc = G.model(**{k: getattr(c, k) for k in ("dim", "heads", "kv", "layers", "eps", "theta", "vocab", "ffn", "places", "rope", "tied")})
  w = None if share is not None else G.numpy_weights(OL.random_weights(c, np.random.default_rng(seed)))
  return G.Decoder(gc, w, mode="bfp8", kv=kv, batch=batch, context=context, slots=slots, share=share, mfma_from=mfma_from)


def close(got, want, what):
  got, want = got.double().cpu(), want.double().cpu()
  rel = float((got - want).abs().max() / want.abs().max())
  cos = float((got * want).sum() / (got.norm() * want.norm()))
  assert rel <= 1e-2 and cos >= 0.9999, (what, rel, cos)


@pytest.mark.parametrize("kv", ["bf16", "bfp8", "fp32"])
@pytest.mark.parametrize("n,mfma_from", [(5, 3), (2, None)])
def test_shared_prefix_end_to_end(cuda, kv, n, mfma_from):
  rng = np.random.default_rng(61)
  system = [int(i) for i in rng.integers(0, 2048, SYSTEM)]
  prompts = [[int(i) for i in rng.integers(0, 2048, m)] for m in PROMPTS[:n]]
  whole = decoder(62, kv, n, 200, n, mfma_from=mfma_from)
  want = torch.cat([whole.prefill(system + p, slot=i)[0].clone() for i, p in enumerate(prompts)])
  dec = decoder(62, kv, n, 100, n + 1, share=whole, mfma_from=mfma_from)
  dec.prefill(system, slot=n)
  dec.share_prefix(n, SYSTEM)
  got, picks = dec.prefill_batch(prompts)
  close(got, want, "prompts' logits")
  assert torch.equal(picks.long().cpu(), got.argmax(1).cpu())
  nxt = [int(i) for i in rng.integers(0, 2048, n)]
  places = [SYSTEM + len(p) for p in prompts]
  for step in range(4):
    if step < 2:
      a, b = whole.step(nxt, places, list(range(n)))[0], dec.step(nxt, places, list(range(n)))[0]
      places = [p + 1 for p in places]
    else:  # (the next tokens the first decoder's picks, on the GPU)
      whole.advance()
      dec.advance()
      dec.ids.copy_(whole.ids)
      a, b = whole.step()[0], dec.step()[0]
    close(b, a, ("step", step))


def test_rows_that_share_less_or_nothing(cuda):
  # a batch in which one row shares half the prefix and one none of it, then the sharing ends and the slots are whole again
  rng = np.random.default_rng(63)
  system = [int(i) for i in rng.integers(0, 2048, SYSTEM)]
  prompts = [[int(i) for i in rng.integers(0, 2048, m)] for m in (20, 7, 40)]
  sh = [SYSTEM, SYSTEM // 2, 0]
  whole = decoder(64, "bf16", 3, 200, 3)
  want = torch.cat([whole.prefill(system[:s] + p, slot=i)[0].clone() for i, (s, p) in enumerate(zip(sh, prompts))])
  dec = decoder(64, "bf16", 3, 120, 4, share=whole)
  dec.prefill(system, slot=3)
  dec.share_prefix(3, SYSTEM, rows=sh)
  close(dec.prefill_batch(prompts, shared=sh)[0], want, "prompts")
  places = [s + len(p) for s, p in zip(sh, prompts)]
  close(dec.step([1, 2, 3], places, [0, 1, 2])[0], whole.step([1, 2, 3], places, [0, 1, 2])[0], "step")
  # a second turn behind what is cached: prompts at later places
  more = [[int(i) for i in rng.integers(0, 2048, m)] for m in (3, 30)]
  got = dec.prefill_batch(more, slots=[2, 0], p0=[places[2] + 1, places[0] + 1], shared=[0, SYSTEM])[0]
  want = torch.cat([whole.prefill(m, slot=i, p0=places[i] + 1)[0].clone() for m, i in zip(more, (2, 0))])
  close(got, want, "second turn")
  dec.share_prefix()
  dec.prefill(prompts[2], slot=0)
  close(dec.step([5, 5, 5], [len(prompts[2])] * 3, [0, 0, 0], replay=True)[0], whole_step(whole, prompts[2]), "no sharing")


def whole_step(whole, prompt):
  whole.prefill(prompt, slot=0)
  return whole.step([5, 5, 5], [len(prompt)] * 3, [0, 0, 0])[0]


def test_unshared_packed_prompts_fill_the_cache_as_prefill_does(cuda):
  rng = np.random.default_rng(65)
  prompts = [[int(i) for i in rng.integers(0, 2048, m)] for m in (100, 1, 37, 128)]
  one = decoder(66, "bf16", 1, 130, 6)
  want = torch.cat([one.prefill(p, slot=s)[0].clone() for p, s in zip(prompts, (5, 0, 2, 3))])
  many = decoder(66, "bf16", 1, 130, 6, share=one)
  close(many.prefill_batch(prompts, slots=[5, 0, 2, 3])[0], want, "logits")
  for l in range(2):
    close(many.cache[l].float(), one.cache[l].float(), ("cache", l))
    assert (many.cache[l][:, 130:260] == 0).all() and (many.cache[l][:, 520:650] == 0).all()  # (the other slots' rows untouched)


def test_heads_under_rules(cuda):
  # three steps of a batch whose histories grow, each step's heads those of numpy on the step's logits under the rules
  rng = np.random.default_rng(67)
  dec = decoder(68, "bf16", 3, 64, 3)
  V, hist = 2048, torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
  lens = torch.zeros(3, dtype=torch.int32, device="cuda")
  rep, pre, fre = (torch.tensor(v, device="cuda") for v in ([1.3, 1.0, 1.1], [0.0, 0.5, 0.2], [0.1, 0.0, 0.3]))
  allowed = torch.from_numpy(rng.integers(-(1 << 31), 1 << 31, (3, V // 32)).astype(np.int32)).cuda()
  ids, bias = torch.tensor([[7, 9], [-1, 3], [100, 100]], dtype=torch.int32, device="cuda"), torch.tensor([[50.0, -3.0], [9.0, 2.0], [1.0, 1.5]], device="cuda")
  tokens, at = torch.tensor([4, 8, 15], dtype=torch.int32, device="cuda"), 0
  for step in range(3):
    hist[:, step] = tokens
    lens += 1
    logits = dec.step(tokens, [step] * 3, [0, 1, 2])[0].clone()
    values, picks, lse = dec.heads(8, [1.0, 0.5, 2.0], rules=dict(tokens=hist, lengths=lens, repetition=rep, presence=pre, frequency=fre, bias_ids=ids,
                                                                 bias=bias, allowed=allowed))
    assert torch.equal(dec.logits, logits)  # (the step's own are as they were)
    x = logits.double().cpu().numpy()
    for r in range(3):
      seen, n = np.unique(hist[r, :step + 1].cpu().numpy(), return_counts=True)
      x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / float(rep[r]), x[r, seen] * float(rep[r]))
      x[r, seen] -= float(fre[r]) * n + float(pre[r])
      for i, b in zip(ids[r].tolist(), bias[r].tolist()):
        if i >= 0: x[r, i] += b
      bits = (allowed[r].cpu().numpy().view(np.uint32)[np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32)) & 1
      x[r, bits == 0] = -np.inf
      wv, _, wl = head_of(x[r].astype(np.float32), [1.0, 0.5, 2.0][r], 8)
      v = values[r].cpu().numpy()
      assert (np.abs(v - wv) <= 8 * 2.0 ** -24 * np.abs(wv) + 1e-30).all() and abs(float(lse[r]) - wl) <= 1e-5 * abs(wl) + 1e-5
      assert (np.abs(x[r][picks[r].cpu().numpy()] - v) <= 8 * 2.0 ** -24 * np.abs(v)).all()
    tokens = picks[:, 0].contiguous()
  plain = dec.heads(4)
  assert torch.equal(plain[1][:, 0].long(), dec.logits.argmax(1))


def test_refusals(cuda):
  dec = decoder(69, "bf16", 2, 64, 3)
  for kw in (dict(slot=3, length=4), dict(slot=0, length=0), dict(slot=0, length=65), dict(slot=0, length=4, rows=[5, 0]), dict(slot=0, length=4, rows=[1])):
    with pytest.raises(ValueError): dec.share_prefix(**kw)
  with pytest.raises(ValueError): dec.prefill_batch([])
  with pytest.raises(ValueError): dec.prefill_batch([[1], []])
  with pytest.raises(ValueError): dec.prefill_batch([[1], [2]], slots=[1, 1])
  with pytest.raises(ValueError): dec.prefill_batch([[1] * 65])
  with pytest.raises(ValueError): dec.prefill_batch([[1]], shared=[3])
  dec.prefill([1, 2, 3], slot=2)
  dec.share_prefix(2, 3)
  with pytest.raises(ValueError): dec.step()                       # (the rows' places are those of before)
  with pytest.raises(ValueError): dec.prefill([1], slot=0)
  with pytest.raises(ValueError): dec.prefill_batch([[1]], slots=[2])
  with pytest.raises(ValueError): dec.prefill_batch([[1]], p0=[2])
  with pytest.raises(ValueError): dec.set_rows([2, 3], [0, 1])      # (place 2 is the prefix's)
  with pytest.raises(ValueError): dec.set_rows([3, 3], [0, 2])      # (slot 2 is the prefix's)
  with pytest.raises(ValueError): dec.set_rows([3, 67], [0, 1])
  dec.step([1, 2], [3, 66], [0, 1])
  with pytest.raises(ValueError): dec.advance()
