"""The operators of a service that runs many requests at once, as cases to time and check: causal attention over packed
prompts (attention_prefill_packed), decode attention of a batch that shares a prefix (attention_decode_shared), and each
request's penalties, biases and grammar mask on its logits (logit_rules). listed() names the cases, draw() gives more of
the same ranges, prepare() makes what a program holds before the call, run() is one pass (the framework's where `own` is
true, plain torch otherwise), and exact() the same outputs in 64 bits."""
import math
import random
import torch

own = False
DEV = "cuda"

# heads, key heads and head_dim of the models the framework is measured on (SmolLM-135M, Llama-3.1-8B and a generic one)
HEADS = {"smollm-135m": (9, 3, 64), "llama-8b": (32, 8, 128), "generic-2k": (32, 8, 64)}
VOCAB = {"smollm-135m": 49152, "llama-8b": 128256, "generic-2k": 32000}
DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
  return [
    # the smallest call: three one-line questions to a small model, latency alone
    dict(name="packed smollm 3x20", kind="packed", model="smollm-135m", n=3, longest=20, cached=0, prefix=0, spread=1, pad=4, q="fp32", kv="bf16", o="bf16"),
    # a service's ordinary step of prompts: 16 chat turns of up to 400 tokens
    dict(name="packed 8b 16x400", kind="packed", model="llama-8b", n=16, longest=400, cached=0, prefix=0, spread=2, pad=0, q="fp32", kv="bf16", o="bf16"),
    # long documents: four of up to 4096 tokens, q as a bf16 model holds it
    dict(name="packed 8b 4x4096", kind="packed", model="llama-8b", n=4, longest=4096, cached=0, prefix=0, spread=3, pad=64, q="bf16", kv="bf16", o="bf16"),
    # questions of up to 130 tokens behind one system prompt of 1500, some after turns of their own, in a block-float cache
    dict(name="packed 2k 24x130 after 1500", kind="packed", model="generic-2k", n=24, longest=130, cached=90, prefix=1500, spread=4, pad=16, q="fp32",
         kv="bfp8", o="bf16"),
    # a check of a small model in full precision
    dict(name="packed smollm 6x300 fp32", kind="packed", model="smollm-135m", n=6, longest=300, cached=0, prefix=0, spread=5, pad=0, q="fp32", kv="fp32", o="fp32"),
    # four users of a small model behind a short system prompt, a token each, fp32 rows out
    dict(name="shared smollm b4 180", kind="shared", model="smollm-135m", batch=4, prefix=180, longest=40, some=False, spread=1, q="fp32", kv="bf16", o="fp32"),
    # an ordinary service: 16 users behind a system prompt with its tools, 4096 tokens
    dict(name="shared 8b b16 4096", kind="shared", model="llama-8b", batch=16, prefix=4096, longest=300, some=False, spread=2, q="fp32", kv="bf16", o="bf16"),
    # many questions about one long document
    dict(name="shared 8b b64 16384", kind="shared", model="llama-8b", batch=64, prefix=16384, longest=700, some=False, spread=3, q="fp32", kv="bf16", o="bf16"),
    # rows that branched off a long prompt at places of their own, some not at all, in a bfp4 cache
    dict(name="shared 2k b23 6001 some", kind="shared", model="generic-2k", batch=23, prefix=6001, longest=500, some=True, spread=4, q="fp32", kv="bfp4", o="bf16"),
    # one user's next token
    dict(name="rules smollm b1", kind="rules", vocab=49152, rows=1, history=300, biases=0, mask=False, spread=1),
    # 16 users, some under a grammar, with a few biases; a vocabulary whose rows are not 16-byte aligned
    dict(name="rules 50257 b16 masks", kind="rules", vocab=50257, rows=16, history=2000, biases=20, mask=True, spread=2),
    # a large batch with long histories and lists of biases
    dict(name="rules 8b b128 masks", kind="rules", vocab=128256, rows=128, history=8000, biases=300, mask=True, spread=3),
  ]


def _log(rng, lo, hi):
  return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
  kind = rng.choice(["packed", "shared", "rules"])
  spread = rng.randrange(1 << 20)
  if kind == "rules":
    rows = _log(rng, 1, 128)
    return dict(kind=kind, vocab=rng.choice([_log(rng, 1000, 160000), 49152, 128256, 32000, 50257]) if rows < 100 else _log(rng, 1000, 120000),
                rows=rows, history=rng.choice([0, _log(rng, 1, 8000), _log(rng, 1, 8000)]), biases=rng.choice([0, _log(rng, 1, 300)]),
                mask=rng.random() < 0.6, spread=spread)
  model = rng.choice(list(HEADS))
  kv = rng.choice(["bf16", "bf16", "bfp8", "bfp4", "fp32"])
  q, o = rng.choice(["fp32", "fp32", "bf16"]), rng.choice(["bf16", "bf16", "fp32"])
  if kind == "packed":
    longest = _log(rng, 1, 2048 if kv != "fp32" and o == "bf16" else 700)
    n = _log(rng, 1, max(1, min(64, 8000 // (longest + 60))))
    return dict(kind=kind, model=model, n=n, longest=longest, cached=rng.choice([0, 0, _log(rng, 1, 1500)]),
                prefix=rng.choice([0, 0, _log(rng, 1, 2000)]), spread=spread, pad=rng.choice([0, rng.randrange(1, 80)]), q=q, kv=kv, o=o)
  batch = _log(rng, 1, 64)
  return dict(kind=kind, model=model, batch=batch, prefix=_log(rng, 1, 16000 if kv != "fp32" and o == "bf16" else 4000),
              longest=_log(rng, 1, 700), some=rng.random() < 0.4, spread=spread, q=q, kv=kv, o=o)


# ---- the shapes of a case: by the case alone ---------------------------------------------------------------------------
def _packed_shape(case):
  """Each prompt's tokens, cached places before them (behind the prefix) and first own cache row; the cache's rows."""
  rng = random.Random(case["spread"])
  lens = [max(0, round(case["longest"] * rng.uniform(0.25, 1.0))) or 1 for _ in range(case["n"])]
  lens[rng.randrange(case["n"])] = case["longest"]
  if case["n"] > 4: lens[rng.randrange(case["n"])] = 0  # (a request cancelled after its place in the batch was given)
  cached = [rng.choice([0, rng.randrange(case["cached"] + 1)]) for _ in range(case["n"])]
  first, at = [], case["prefix"] + 3
  for a, b in zip(lens, cached):
    first.append(at)
    at += a + b + rng.randrange(4)
  return lens, cached, first, at + 1


def _shared_shape(case):
  """Each row's prefix rows, own rows and first own cache row; the cache's rows."""
  rng = random.Random(case["spread"])
  B, P = case["batch"], case["prefix"]
  shared = [P] * B
  mine = [1 + rng.randrange(case["longest"]) for _ in range(B)]
  mine[rng.randrange(B)] = case["longest"]
  if case["some"]:
    shared = [rng.choice([P, P, 0, rng.randrange(P + 1)]) for _ in range(B)]
    if B > 2: shared[rng.randrange(B)] = P
    if B > 3: shared[1], mine[1] = 0, 0  # (a row of the batch that no request holds)
  first = []
  at = P + 5
  for m in mine:
    first.append(at)
    at += m + rng.randrange(3)
  return shared, mine, first, at + 1


def _gen(seed, name):
  g = torch.Generator(device=DEV)
  g.manual_seed((seed * 1000003 + sum(ord(c) * 31 ** i for i, c in enumerate(name))) % (1 << 62))
  return g


def _normal(seed, name, shape, sd=1.0, dtype=torch.float32):
  return (torch.randn(*shape, generator=_gen(seed, name), device=DEV) * sd).to(dtype)


def _whole(seed, name, lo, hi, shape):
  return torch.randint(lo, hi, shape, generator=_gen(seed, name), device=DEV, dtype=torch.int32)


def _ints(values):
  return torch.tensor(values, dtype=torch.int32, device=DEV)


def _cache(seed, planes, rows, hd, kv):
  """Keys' heads then values': a tensor, or a block float's one buffer (every row's magnitudes, then every row's
  exponents, a byte a run of 16)."""
  x = _normal(seed, "cache", (planes, rows, hd), 1.0, torch.bfloat16)
  if kv in DTYPE: return _normal(seed, "cache", (planes, rows, hd)) if kv == "fp32" else x
  runs = x.float().view(planes * rows, hd // 16, 16)
  top = torch.frexp(runs.abs().amax(2).clamp(min=1e-30)).exponent + 126  # (the run's largest biased exponent)
  if kv == "bfp8":
    m = torch.ldexp(runs, (133 - top)[..., None]).round().clamp(-127, 127).to(torch.int8).view(torch.uint8).reshape(-1)
  else:
    m = torch.ldexp(runs, (129 - top)[..., None]).round().clamp(-7, 7).to(torch.int8).view(torch.uint8).view(-1, 2) & 15
    m = m[:, 0] | (m[:, 1] << 4)
  return torch.cat([m.reshape(-1), top.to(torch.uint8).reshape(-1)])


def prepare(case, seed):
  if case["kind"] == "rules":
    rng = random.Random(case["spread"])
    R, V, H, nb = case["rows"], case["vocab"], case["history"], case["biases"]
    st = dict(logits=_normal(seed, "logits", (R, V), 3.0), out=torch.zeros(R, V, device=DEV), tokens=None, lengths=None, prompts=None,
              bias_ids=None, bias=None, allowed=None)
    if H:
      lens = [rng.randrange(H // 2, H + 1) for _ in range(R)]
      # (a text's tokens: a few hundred common ones again and again, the rest anywhere; -1 past a row's end)
      tok = torch.where(_whole(seed, "common", 0, 3, (R, H)) > 0, _whole(seed, "few", 0, min(V, 400), (R, H)), _whole(seed, "any", 0, V, (R, H)))
      st["lengths"], st["prompts"] = _ints(lens), _ints([rng.randrange(n + 1) for n in lens])
      st["tokens"] = torch.where(torch.arange(H, device=DEV)[None] < st["lengths"][:, None], tok, -1)
    st["repetition"] = 1.0 + 0.1 * _whole(seed, "rep", 0, 4, (R,)).float()
    st["presence"], st["frequency"] = 0.25 * _whole(seed, "pre", 0, 5, (R,)).float(), 0.1 * _whole(seed, "fre", 0, 5, (R,)).float()
    if nb:
      used = _ints([rng.randrange(nb + 1) for _ in range(R)])
      ids = _whole(seed, "ids", 0, V, (R, nb))
      st["bias_ids"] = torch.where(torch.arange(nb, device=DEV)[None] < used[:, None], ids, -1)
      st["bias"] = _normal(seed, "bias", (R, nb), 4.0)
    if case["mask"]:
      words = _whole(seed, "mask", -(1 << 31), (1 << 31) - 1, (R, -(-V // 32))) & _whole(seed, "mask2", -(1 << 31), (1 << 31) - 1, (R, -(-V // 32)))
      free = _ints([rng.randrange(2) for _ in range(R)])  # (half the rows under no grammar)
      st["allowed"] = torch.where(free[:, None] > 0, torch.full_like(words, -1), words)
    return st
  heads, kv, hd = HEADS[case["model"]]
  if case["kind"] == "packed":
    lens, cached, first, rows = _packed_shape(case)
    T = max(1, sum(lens) + case["pad"])
    starts = [0]
    for n in lens: starts.append(starts[-1] + n)
    st = dict(starts=_ints(starts), p0=_ints([case["prefix"] + c for c in cached]), first=_ints(first), rows=rows, used=starts[-1],
              shared=_ints([case["prefix"]] * case["n"]) if case["prefix"] else None, longest=case["longest"],
              context=case["prefix"] + max(a + b for a, b in zip(lens, cached)))
  else:
    shared, mine, first, rows = _shared_shape(case)
    T = case["batch"]
    st = dict(shared=_ints(shared), places=_ints([a + b - 1 for a, b in zip(shared, mine)]), first=_ints(first), rows=rows, prefix=case["prefix"],
              longest=case["longest"])
  st["cache"] = _cache(seed, 2 * kv, rows, hd, case["kv"])
  st["prefix_row"] = _ints([2])
  st["q"] = _normal(seed, "q", (T, heads * hd), 1.5, DTYPE[case["q"]])
  st["o"] = torch.zeros(T, heads * hd, dtype=DTYPE[case["o"]], device=DEV)
  st["case"] = case
  return st


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _own_run(st):
  from ferrite_amd import ops
  if "logits" in st:
    return ops.logit_rules(st["logits"], tokens=st["tokens"], lengths=st["lengths"], prompt_lengths=st["prompts"], repetition=st["repetition"],
                           presence=st["presence"], frequency=st["frequency"], bias_ids=st["bias_ids"], bias=st["bias"], allowed=st["allowed"], out=st["out"])
  case = st["case"]
  heads, kv, hd = HEADS[case["model"]]
  cache = st["cache"] if case["kv"] in DTYPE else ops.BfpCache(st["cache"], case["kv"], 2 * kv, st["rows"], hd)
  if case["kind"] == "packed":
    if "ws" not in st: st["ws"] = ops.attention_packed_workspace(st["q"].shape[0], case["n"], heads, kv, hd, st["context"])
    prefix = dict(prefix_row=st["prefix_row"], shared=st["shared"]) if case["prefix"] else {}
    return ops.attention_prefill_packed(st["q"], cache, heads, kv, hd, st["starts"], st["p0"], st["first"], st["context"], workspace=st["ws"], o=st["o"], **prefix)
  if "ws" not in st: st["ws"] = ops.attention_shared_workspace(case["batch"], heads, kv, hd, st["prefix"], st["longest"])
  return ops.attention_decode_shared(st["q"], cache, heads, kv, hd, st["places"], st["first"], st["prefix_row"], st["shared"], st["prefix"], st["longest"],
                                     workspace=st["ws"], o=st["o"])


# ---- the plain forms: 32 bits, rounded once ----------------------------------------------------------------------------
def _values(st, case, planes, hd):
  """The cache's values in 32 bits."""
  if case["kv"] in DTYPE: return st["cache"].float()
  n = planes * st["rows"]
  width = hd if case["kv"] == "bfp8" else hd // 2
  m, e = st["cache"][:n * width].view(n, width), st["cache"][n * width:].view(n, hd // 16, 1)
  if case["kv"] == "bfp4": m = torch.stack([m << 4, m & 240], 2)  # (16 q: a byte's upper half)
  v = m.reshape(n, hd // 16, 16).view(torch.int8).float()
  return (v * torch.exp2(e.float() - 133.0)).view(planes, st["rows"], hd)


def _plain_packed(st):
  case = st["case"]
  heads, kv, hd = HEADS[case["model"]]
  n, L, K, rep = case["n"], st["longest"], st["context"], heads // kv
  lens = st["starts"][1:] - st["starts"][:-1]
  t, p = torch.arange(L, device=DEV), torch.arange(K, device=DEV)
  here = t[None] < lens[:, None]                                                     # [n][L]: the prompts padded to the longest
  at = (st["starts"][:-1, None] + t[None]).clamp(max=st["q"].shape[0] - 1)
  sh = st["shared"] if st["shared"] is not None else torch.zeros_like(lens)
  row = torch.where(p[None] < sh[:, None], st["prefix_row"] + p[None], st["first"][:, None] + p[None] - sh[:, None]).clamp(0, st["rows"] - 1)
  k, v = _values(st, case, 2 * kv, hd)[:, row].transpose(0, 1).split(kv, 1)            # [n][kv][K][hd]
  q = st["q"][at].float().view(n, L, kv, rep, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, rep * L, hd)
  s = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(hd)).view(n, kv, rep, L, K)
  s.masked_fill_((p[None, None] > (st["p0"][:, None] + t[None])[..., None])[:, None, None], -math.inf)
  s = s.sub_(s.amax(-1, keepdim=True)).exp_()
  s = s.div_(s.sum(-1, keepdim=True)).view(n, kv, rep * L, K)
  o = torch.matmul(s, v).view(n, kv, rep, L, hd).permute(0, 3, 1, 2, 4).reshape(n, L, heads * hd)
  st["o"][:st["used"]] = o[here].to(st["o"].dtype)
  return st["o"]


def _plain_shared(st):
  case = st["case"]
  heads, kv, hd = HEADS[case["model"]]
  B, P, M, rep = case["batch"], st["prefix"], st["longest"], heads // kv
  c = _values(st, case, 2 * kv, hd)
  p, m = torch.arange(P, device=DEV), torch.arange(M, device=DEV)
  k0, v0 = c[:, st["prefix_row"] + p].split(kv, 0)                                     # [kv][P][hd]: once for the batch
  k1, v1 = c[:, (st["first"][:, None] + m[None]).clamp(max=st["rows"] - 1)].transpose(0, 1).split(kv, 1)  # [B][kv][M][hd]
  q = st["q"].float().view(B, kv, rep, hd)
  s0 = torch.matmul(q.transpose(0, 1).reshape(kv, B * rep, hd), k0.transpose(-1, -2)).view(kv, B, rep, P).transpose(0, 1)
  s = torch.cat([s0, torch.matmul(q, k1.transpose(-1, -2))], -1) / math.sqrt(hd)      # [B][kv][rep][P + M]
  seen = torch.cat([p[None] < torch.minimum(st["shared"], st["places"] + 1)[:, None], m[None] <= (st["places"] - st["shared"])[:, None]], 1)[:, None, None]
  s = s.masked_fill(~seen, -math.inf)
  e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))                       # (a row that sees nothing: zeros)
  e = e / e.sum(-1, keepdim=True).clamp(min=1e-30)
  o = torch.matmul(e[..., :P].transpose(0, 1).reshape(kv, B * rep, P), v0).view(kv, B, rep, hd).transpose(0, 1) + torch.matmul(e[..., P:], v1)
  st["o"].copy_(o.reshape(B, heads * hd))
  return st["o"]


def _plain_rules(st):
  x = st["logits"]
  R, V = x.shape
  y = x
  if st["tokens"] is not None:
    j = torch.arange(st["tokens"].shape[1], device=DEV)[None]
    inside = (j < st["lengths"][:, None]) & (st["tokens"] >= 0)
    at = torch.where(inside, st["tokens"], V).long()
    ones = torch.ones_like(at, dtype=torch.float32)
    seen = torch.zeros(R, V + 1, device=DEV).scatter_add_(1, at, ones)[:, :V] > 0
    n = torch.zeros(R, V + 1, device=DEV).scatter_add_(1, at, torch.where(j >= st["prompts"][:, None], ones, 0.0))[:, :V]
    r = st["repetition"][:, None]
    y = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    y = y - st["frequency"][:, None] * n - st["presence"][:, None] * (n > 0)
  if st["bias"] is not None:
    at = torch.where(st["bias_ids"] >= 0, st["bias_ids"], V).long()
    y = y + torch.zeros(R, V + 1, device=DEV).scatter_add_(1, at, st["bias"])[:, :V]
  if st["allowed"] is not None:
    bits = (st["allowed"][..., None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
    y = torch.where(bits.view(R, -1)[:, :V] > 0, y, -math.inf)
  st["out"].copy_(y)
  return st["out"]


def run(st):
  if own: return _own_run(st)
  if "logits" in st: return _plain_rules(st)
  return _plain_packed(st) if st["case"]["kind"] == "packed" else _plain_shared(st)


def work(case):
  if case["kind"] == "rules":
    R, V = case["rows"], case["vocab"]
    n = 8 * R * V + (R * -(-V // 32) * 4 if case["mask"] else 0) + R * case["history"] * 3 + 8 * R * case["biases"]
    return {"bytes": n, "flops": 4 * R * V}
  heads, kv, hd = HEADS[case["model"]]
  row = {"fp32": 4 * hd, "bf16": 2 * hd, "bfp8": hd + hd // 16, "bfp4": hd // 2 + hd // 16}[case["kv"]]
  if case["kind"] == "packed":
    lens, cached, _, _ = _packed_shape(case)
    T, rows = sum(lens), case["prefix"] + sum(a + b for a, b in zip(lens, cached) if a)
    pairs = sum(a * (case["prefix"] + b) + a * (a + 1) // 2 for a, b in zip(lens, cached))
  else:
    shared, mine, _, _ = _shared_shape(case)
    T, rows, pairs = case["batch"], max(shared) + sum(mine), sum(shared) + sum(mine)
  io = T * heads * hd * ((4 if case["q"] == "fp32" else 2) + (4 if case["o"] == "fp32" else 2))
  return {"bytes": 2 * kv * row * rows + io, "flops": 4 * hd * heads * pairs}


# ---- the same in 64 bits: a sequence, a row at a time ------------------------------------------------------------------
def _exact_cache(case, st, planes, hd):
  raw, rows = st["cache"], st["rows"]
  if case["kv"] in DTYPE: return raw.double()
  count = planes * rows * hd
  if case["kv"] == "bfp8": q = raw[:count].to(torch.int64)
  else:
    low = raw[:count // 2].to(torch.int64)
    q = torch.empty(count, dtype=torch.int64, device=DEV)
    q[0::2], q[1::2] = low % 16, low // 16
  span, bias = (256, 133) if case["kv"] == "bfp8" else (16, 129)
  q = torch.where(q >= span // 2, q - span, q).double()
  e = raw[-(count // 16):].to(torch.int64).repeat_interleave(16) - bias
  return torch.ldexp(q, e).view(planes, rows, hd)


def _attend64(q, cache, where, limit, kv, hd):
  """q [L][heads hd] over cache rows `where`, row t seeing the first limit[t] of them."""
  L, rep = q.shape[0], q.shape[1] // hd // kv
  out = torch.zeros(L, kv, rep, hd, dtype=torch.float64, device=DEV)
  hidden = torch.arange(len(where), device=DEV)[None] >= limit[:, None]
  for g in range(kv):
    k, v = cache[g][where], cache[kv + g][where]
    for r in range(rep):
      h = g * rep + r
      s = (q[:, h * hd:(h + 1) * hd].double() @ k.T.contiguous()) / math.sqrt(hd)
      out[:, g, r] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v
  return out.reshape(L, -1)


def exact(case, seed):
  st = prepare(case, seed)
  if case["kind"] == "rules":
    y = st["logits"].double()
    tokens = None if st["tokens"] is None else st["tokens"].long()
    for b in range(case["rows"]):
      if tokens is not None:
        n, p = int(st["lengths"][b]), int(st["prompts"][b])
        hist = tokens[b, :n]
        found = torch.unique(hist)
        x = y[b, found]
        r = st["repetition"][b].double()
        y[b, found] = torch.where(x > 0, x / r, x * r)
        ids, times = torch.unique(hist[p:], return_counts=True)
        y[b, ids] -= st["frequency"][b].double() * times.double() + st["presence"][b].double()
      if st["bias"] is not None:
        some = st["bias_ids"][b] >= 0
        y[b].index_add_(0, st["bias_ids"][b][some].long(), st["bias"][b][some].double())
      if st["allowed"] is not None:
        c = torch.arange(case["vocab"], device=DEV)
        w = st["allowed"][b].long() % (1 << 32)
        y[b, (w[c // 32] // (1 << (c % 32))) % 2 == 0] = -math.inf
    return y
  heads, kv, hd = HEADS[case["model"]]
  cache = _exact_cache(case, st, 2 * kv, hd)
  o = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
  if case["kind"] == "packed":
    lens, cached, first, _ = _packed_shape(case)
    at, P = 0, case["prefix"]
    for n, c, f in zip(lens, cached, first):
      if n:
        where = torch.cat([2 + torch.arange(P, device=DEV), f + torch.arange(c + n, device=DEV)])
        o[at:at + n] = _attend64(st["q"][at:at + n], cache, where, P + c + 1 + torch.arange(n, device=DEV), kv, hd)
      at += n
    return o
  shared, mine, first, _ = _shared_shape(case)
  for b, (p, m, f) in enumerate(zip(shared, mine, first)):
    if p + m:
      where = torch.cat([2 + torch.arange(p, device=DEV), f + torch.arange(m, device=DEV)])
      o[b:b + 1] = _attend64(st["q"][b:b + 1], cache, where, torch.tensor([p + m], device=DEV), kv, hd)
  return o
