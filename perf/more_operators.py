"""The operators of a service whose sequences keep their keys and values in pages and whose requests bring adapters, as cases
to time and check: the heads' norms, the rotation and the put into a paged cache in one pass (rope_append_paged), attention of
ragged rows over that cache, prompts and single tokens together (attention_paged), and each row's low-rank adapter beside a
shared projection (lora). listed() names the cases, draw() gives more of the same ranges, prepare() makes what a program holds
before the call, run() is one pass (the framework's where `own` is true, plain torch otherwise), and exact() the same outputs
in 64 bits."""
import math
import random
import torch

own = False
DEV = "cuda"

# dim, heads, key heads, head_dim and the MLP's width (SmolLM-135M and Llama-3.1-8B, which the framework is measured on, and a generic one)
MODELS = {"smollm-135m": (576, 9, 3, 64, 1536), "llama-8b": (4096, 32, 8, 128, 14336), "generic-1k": (1280, 20, 4, 64, 3456)}
DTYPE = {"fp32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
  return [
    # the smallest call: one user's next token of a small model
    dict(name="append smollm b1", kind="append", model="smollm-135m", n=1, longest=1, single=1.0, context=200, page=64, norm=False, spread=1, pad=0,
         x="fp32", kv="bf16", q="fp32"),
    # a service's ordinary step: chunks of prompts and single tokens together, rows as a bf16 projection leaves them, q's and k's heads normed
    dict(name="append 8b mixed 40x300", kind="append", model="llama-8b", n=40, longest=300, single=0.6, context=3000, page=16, norm=True, spread=2, pad=24,
         x="bf16", kv="bf16", q="bf16"),
    # prompts of a generic model into a block-float cache
    dict(name="append 1k 9x500 bfp8", kind="append", model="generic-1k", n=9, longest=500, single=0.0, context=100, page=32, norm=True, spread=3, pad=5,
         x="fp32", kv="bfp8", q="fp32"),
    # four users of a small model, a token each, fp32 rows out
    dict(name="paged smollm b4 300", kind="paged", model="smollm-135m", n=4, longest=1, single=1.0, context=300, page=64, spread=1, pad=0, q="fp32",
         kv="bf16", o="fp32"),
    # an ordinary decode step: 16 users at places of their own up to 2000, small pages
    dict(name="paged 8b b16 2000", kind="paged", model="llama-8b", n=16, longest=1, single=1.0, context=2000, page=16, spread=2, pad=0, q="fp32",
         kv="bf16", o="bf16"),
    # a large decode step with long conversations
    dict(name="paged 8b b48 8000", kind="paged", model="llama-8b", n=48, longest=1, single=1.0, context=8000, page=64, spread=3, pad=0, q="bf16",
         kv="bf16", o="bf16"),
    # a step of a service that cuts its prompts in chunks: single tokens and chunks of up to 512 in one call
    dict(name="paged 8b mixed 24x512", kind="paged", model="llama-8b", n=24, longest=512, single=0.7, context=4000, page=16, spread=4, pad=8, q="bf16",
         kv="bf16", o="bf16"),
    # a generic model's prompts after earlier turns, in a block-float cache
    dict(name="paged 1k 11x250 bfp8", kind="paged", model="generic-1k", n=11, longest=250, single=0.2, context=900, page=32, spread=5, pad=3, q="fp32",
         kv="bfp8", o="bf16"),
    # one user's adapter beside q, k and v of a small model, for a token
    dict(name="lora smollm qkv b1", kind="lora", model="smollm-135m", at="qkv", rank=8, adapters=1, rows=1, prompts=0, none=0.0, spread=1, x="fp32",
         w="bf16", y="fp32"),
    # a decode step of 32 users, each with one of 24 adapters, a few with none
    dict(name="lora 8b qkv b32", kind="lora", model="llama-8b", at="qkv", rank=16, adapters=24, rows=32, prompts=0, none=0.1, spread=2, x="bf16",
         w="bf16", y="fp32"),
    # prompts of eight requests with four adapters, packed, beside gate and up
    dict(name="lora 8b gate_up 4096", kind="lora", model="llama-8b", at="gate_up", rank=32, adapters=4, rows=4096, prompts=8, none=0.0, spread=3, x="bf16",
         w="bf16", y="bf16"),
    # full precision, an odd rank and odd prompts, some rows with no adapter
    dict(name="lora 1k down 333 fp32", kind="lora", model="generic-1k", at="down", rank=20, adapters=6, rows=333, prompts=9, none=0.25, spread=4, x="fp32",
         w="fp32", y="fp32"),
  ]


def _log(rng, lo, hi):
  return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
  kind = rng.choice(["append", "paged", "lora"])
  spread = rng.randrange(1 << 20)
  model = rng.choice(list(MODELS))
  if kind == "lora":
    rows = _log(rng, 1, 3500)
    tokens = rows <= 64 and rng.random() < 0.7
    wide = rng.random() < 0.5
    return dict(kind=kind, model=model, at=rng.choice(["qkv", "o", "gate_up", "down"]), rank=_log(rng, 1, 64) if rows < 2000 else _log(rng, 1, 32),
                adapters=_log(rng, 1, 24 if rows < 300 else 6), rows=rows, prompts=0 if tokens else _log(rng, 1, min(rows, 12)),
                none=rng.choice([0.0, 0.0, 0.2]), spread=spread, x="fp32" if wide else "bf16", w=rng.choice(["bf16", "bf16", "fp32"]) if wide else "bf16",
                y="fp32" if wide and rows < 1500 else rng.choice(["bf16", "fp32"]) if rows < 1500 else "bf16")
  page = rng.choice([16, 16, 32, 64, 128])
  pad = rng.choice([0, 0, rng.randrange(1, 40)])
  single = rng.choice([1.0, 1.0, 0.0, rng.random()])
  longest = 1 if single == 1.0 else _log(rng, 2, 600)
  n = _log(rng, 1, 64 if single == 1.0 else max(1, min(40, 6000 // (longest + 50))))
  if kind == "append":
    return dict(kind=kind, model=model, n=n, longest=longest, single=single, context=_log(rng, 1, 2000), page=page, norm=rng.random() < 0.5, spread=spread,
                pad=pad, x=rng.choice(["fp32", "bf16"]), kv=rng.choice(["bf16", "bf16", "fp32", "bfp8"]), q=rng.choice(["fp32", "bf16"]))
  kv = rng.choice(["bf16", "bf16", "bfp8", "bfp4", "fp32"])
  o = rng.choice(["bf16", "bf16", "fp32"])
  return dict(kind=kind, model=model, n=min(n, 48), longest=longest, single=single, context=_log(rng, 1, 8000 if single == 1.0 and kv != "fp32" else 3000),
              page=page, spread=spread, pad=pad, q=rng.choice(["fp32", "bf16"]), kv=kv, o=o)


# ---- the shapes of a case: by the case alone ---------------------------------------------------------------------------
def _shape(case):
  """Each sequence's query rows, places before them and pages; the cache's pages."""
  rng = random.Random(case["spread"])
  n = case["n"]
  lens = [1 if rng.random() < case["single"] else max(1, round(case["longest"] * rng.uniform(0.25, 1.0))) for _ in range(n)]
  before = [round(case["context"] * rng.uniform(0.1, 1.0)) for _ in range(n)]
  lens[0], before[-1] = case["longest"], case["context"]
  if n > 2: before[1] = 0                      # (a new conversation)
  if n > 4: lens[rng.randrange(1, n)] = 0      # (a request cancelled after its place in the batch was given)
  count = [-(-(a + b) // case["page"]) for a, b in zip(lens, before)]
  pages = list(range(sum(count) + 3))
  rng.shuffle(pages)                           # (pages as they came free: anywhere)
  own_pages, at = [], 0
  for c in count:
    own_pages.append(pages[at:at + c])
    at += c
  return lens, before, own_pages, len(pages)


def _lora_shape(case):
  """The projection's K, its parts' columns, and each row's adapter (-1: none)."""
  dim, heads, kv, hd, ffn = MODELS[case["model"]]
  K, cols = {"qkv": (dim, [heads * hd, kv * hd, kv * hd]), "o": (heads * hd, [dim]), "gate_up": (dim, [ffn, ffn]), "down": (ffn, [dim])}[case["at"]]
  rng = random.Random(case["spread"])
  pick = lambda: -1 if rng.random() < case["none"] else rng.randrange(case["adapters"])
  T, parts = case["rows"], case["prompts"]
  if not parts: return K, cols, [pick() for _ in range(T)]
  cuts = [0] + sorted(rng.randrange(T + 1) for _ in range(parts - 1)) + [T]
  ids = []
  for a, b in zip(cuts, cuts[1:]): ids += [pick()] * (b - a)
  return K, cols, ids


def _gen(seed, name):
  g = torch.Generator(device=DEV)
  g.manual_seed((seed * 1000003 + sum(ord(c) * 31 ** i for i, c in enumerate(name))) % (1 << 62))
  return g


def _normal(seed, name, shape, sd=1.0, dtype=torch.float32):
  return (torch.randn(*shape, generator=_gen(seed, name), device=DEV) * sd).to(dtype)


def _ints(values):
  return torch.tensor(values, dtype=torch.int32, device=DEV)


def _packed(values, fmt):
  """bf16 values [rows][hd] as a block float: each row's magnitudes (uint8) and each run of 16's exponent."""
  bits = values.view(torch.int16).int() & 0xFFFF
  e = (bits >> 7 & 255).view(values.shape[0], -1, 16)
  m = torch.where(e > 0, 128, 0) | (bits & 127).view_as(e)
  top = e.amax(-1, keepdim=True)
  sh = top - e
  if fmt == "bfp8":
    sh = sh.clamp(max=8)
    q = ((m + (1 << sh)) >> (sh + 1)).clamp(max=127)
  else:
    q = torch.where(sh < 4, ((m + (16 << sh)) >> (sh + 5)).clamp(max=7), 0)
  q = torch.where((bits >> 15).view_as(e) > 0, -q, q).view(values.shape).to(torch.int8).view(torch.uint8)
  if fmt == "bfp4": q = (q[:, 0::2] & 15) | (q[:, 1::2] << 4)
  return q, top[..., 0].to(torch.uint8)


def _cache(seed, planes, rows, hd, kv):
  """Keys' heads then values': a tensor, or a block float's one buffer (every row's magnitudes, then every row's exponents)."""
  x = _normal(seed, "cache", (planes, rows, hd), 1.0, torch.bfloat16)
  if kv == "fp32": return _normal(seed, "cache", (planes, rows, hd))
  if kv == "bf16": return x
  m, e = _packed(x.view(planes * rows, hd), kv)
  return torch.cat([m.reshape(-1), e.reshape(-1)])


def prepare(case, seed):
  if case["kind"] == "lora":
    K, cols, ids = _lora_shape(case)
    n, T, S, N, r = case["adapters"], case["rows"], len(cols), sum(cols), case["rank"]
    r8 = -(-r // 8) * 8  # (ranks are kept in eights, zeros behind)
    w = DTYPE[case["w"]]
    a = _normal(seed, "a", (n, S, r8, K), K ** -0.5, w)
    b = _normal(seed, "b", (n, N, r8), 0.5 * r ** -0.5, w)
    a[:, :, r:], b[:, :, r:] = 0, 0
    return dict(case=case, a=a.view(n, S * r8, K), b=b, scale=1.0 + 0.25 * torch.arange(n, device=DEV).float(), cols=cols, rank=r8, ids=_ints(ids),
                x=_normal(seed, "x", (T, K), 1.0, DTYPE[case["x"]]), base=_normal(seed, "y", (T, N), 1.0, DTYPE[case["y"]]),
                y=torch.zeros(T, N, dtype=DTYPE[case["y"]], device=DEV))
  dim, heads, kv, hd, _ = MODELS[case["model"]]
  lens, before, own_pages, pages = _shape(case)
  starts = [0]
  for a in lens: starts.append(starts[-1] + a)
  T, widest = max(1, starts[-1] + case["pad"]), max(1, max(len(p) for p in own_pages))
  st = dict(case=case, starts=_ints(starts), p0=_ints(before), used=starts[-1], rows=pages * case["page"], longest=max(lens),
            most=max(a + b for a, b in zip(lens, before)), tables=_ints([p + [-1] * (widest - len(p)) for p in own_pages]))
  st["cache"] = _cache(seed, 2 * kv, st["rows"], hd, case["kv"])
  if case["kind"] == "append":
    # (a projection's rows: q's, k's and v's heads; the rotation's tables hold bf16 values)
    st["x"] = _normal(seed, "x", (T, (heads + 2 * kv) * hd), 1.5, DTYPE[case["x"]])
    angles = torch.arange(st["most"] + 1, device=DEV).double()[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, device=DEV).double() / hd)[None]
    st["cos"], st["sin"] = (f(angles).to(torch.bfloat16).float().repeat(1, 2).contiguous() for f in (torch.cos, torch.sin))
    st["q_norm"], st["k_norm"] = ((1 + _normal(seed, name, (hd,), 0.1)) if case["norm"] else None for name in ("q_norm", "k_norm"))
    st["q"] = torch.zeros(T, heads * hd, dtype=DTYPE[case["q"]], device=DEV)
  else:
    st["q"] = _normal(seed, "q", (T, heads * hd), 1.5, DTYPE[case["q"]])
    st["o"] = torch.zeros(T, heads * hd, dtype=DTYPE[case["o"]], device=DEV)
  return st


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _own_run(st):
  from ferrite_amd import ops
  case = st["case"]
  if case["kind"] == "lora":
    if "adapters" not in st: st["adapters"] = ops.Adapters(st["a"], st["b"], st["scale"], tuple(st["cols"]))
    if "ws" not in st: st["ws"] = ops.lora_workspace(case["rows"], st["adapters"])
    return ops.lora(st["x"], st["adapters"], st["ids"], residual=st["base"], out=st["y"], workspace=st["ws"])
  dim, heads, kv, hd, _ = MODELS[case["model"]]
  cache = st["cache"] if case["kv"] in DTYPE else ops.BfpCache(st["cache"], case["kv"], 2 * kv, st["rows"], hd)
  if case["kind"] == "append":
    ops.rope_append_paged(st["x"], cache, heads, kv, hd, st["cos"], st["sin"], st["starts"], st["p0"], st["tables"], case["page"], q_norm=st["q_norm"],
                          k_norm=st["k_norm"], eps=EPS, q=st["q"])
    return st["q"], _held(st, case, 2 * kv, hd)
  if "ws" not in st: st["ws"] = ops.attention_paged_workspace(st["q"].shape[0], case["n"], heads, kv, hd, st["most"])
  return ops.attention_paged(st["q"], cache, heads, kv, hd, st["starts"], st["p0"], st["tables"], case["page"], st["most"], workspace=st["ws"], o=st["o"])


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


def _held(st, case, planes, hd):
  """The cache as it is: the buffer, or what a block float's bytes stand for."""
  return st["cache"] if case["kv"] in DTYPE else _values(st, case, planes, hd).to(torch.bfloat16)


def _plain_append(st):
  case = st["case"]
  _, heads, kv, hd, _ = MODELS[case["model"]]
  U = st["used"]
  t = torch.arange(U, device=DEV, dtype=torch.int32)
  s = torch.searchsorted(st["starts"][1:].contiguous(), t, right=True)   # each row's sequence
  place = st["p0"][s] + t - st["starts"][s]
  row = (st["tables"][s, place // case["page"]] * case["page"] + place % case["page"]).long()
  x = st["x"][:U].float().view(U, heads + 2 * kv, hd)
  qk, v = x[:, :heads + kv], x[:, heads + kv:]
  if case["norm"]:
    w = torch.cat([st["q_norm"].expand(heads, hd), st["k_norm"].expand(kv, hd)])
    qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
  c, sn = st["cos"][place][:, None], st["sin"][place][:, None]
  qk = qk * c + torch.cat([-qk[..., hd // 2:], qk[..., :hd // 2]], -1) * sn
  st["q"][:U] = qk[:, :heads].reshape(U, heads * hd).to(st["q"].dtype)
  put = torch.cat([qk[:, heads:], v], 1).transpose(0, 1)                 # [2 kv][U][hd]
  if case["kv"] in DTYPE:
    st["cache"][:, row] = put.to(st["cache"].dtype)
  else:
    m, e = _packed(put.to(torch.bfloat16).reshape(2 * kv * U, hd), case["kv"])
    n = 2 * kv * st["rows"]
    at = m.shape[1] * n
    st["cache"][:at].view(2 * kv, st["rows"], m.shape[1])[:, row] = m.view(2 * kv, U, -1)
    st["cache"][at:].view(2 * kv, st["rows"], hd // 16)[:, row] = e.view(2 * kv, U, -1)
  return st["q"], _held(st, case, 2 * kv, hd)


def _plain_paged(st):
  case = st["case"]
  _, heads, kv, hd, _ = MODELS[case["model"]]
  n, L, P, page, rep = case["n"], st["longest"], st["most"], case["page"], heads // kv
  lens = st["starts"][1:] - st["starts"][:-1]
  t, p = torch.arange(L, device=DEV), torch.arange(P, device=DEV)
  here = t[None] < lens[:, None]                                                      # [n][L]: the rows padded to the longest
  at = (st["starts"][:-1, None] + t[None]).clamp(max=st["q"].shape[0] - 1)
  row = st["tables"][:, p // page].clamp(min=0) * page + p % page                     # [n][P]
  k, v = _values(st, case, 2 * kv, hd)[:, row].transpose(0, 1).split(kv, 1)           # [n][kv][P][hd]
  q = st["q"][at].float().view(n, L, kv, rep, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, rep * L, hd)
  s = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(hd)).view(n, kv, rep, L, P)
  s.masked_fill_((p[None, None] > (st["p0"][:, None] + t[None])[..., None])[:, None, None], -math.inf)
  s = s.sub_(s.amax(-1, keepdim=True)).exp_()
  s = s.div_(s.sum(-1, keepdim=True)).view(n, kv, rep * L, P)
  o = torch.matmul(s, v).view(n, kv, rep, L, hd).permute(0, 3, 1, 2, 4).reshape(n, L, heads * hd)
  st["o"][:st["used"]] = o[here].to(st["o"].dtype)
  return st["o"]


def _plain_lora(st):
  n, T, r, cols = st["a"].shape[0], st["x"].shape[0], st["rank"], st["cols"]
  S = len(cols)
  weight = torch.where(st["ids"][:, None] == torch.arange(n, device=DEV), st["scale"], 0.0)  # [T][n]: a row's adapter's scale
  u = torch.matmul(st["x"].float(), st["a"].float().view(n * S * r, -1).T).view(T, n, S, r) * weight[:, :, None, None]
  b = st["b"].float().split(cols, 1)                                                         # each part's [n][columns][r]
  d = [torch.matmul(u[:, :, i].reshape(T, n * r), b[i].transpose(1, 2).reshape(n * r, cols[i])) for i in range(S)]
  st["y"].copy_(st["base"].float() + torch.cat(d, 1))
  return st["y"]


def run(st):
  if own: return _own_run(st)
  return {"lora": _plain_lora, "append": _plain_append, "paged": _plain_paged}[st["case"]["kind"]](st)


_BYTES = {"fp32": 4, "bf16": 2}


def work(case):
  if case["kind"] == "lora":
    K, cols, ids = _lora_shape(case)
    N, S, r = sum(cols), len(cols), case["rank"]
    some, used = sum(i >= 0 for i in ids), len({i for i in ids if i >= 0})
    return {"bytes": some * K * _BYTES[case["x"]] + used * (S * r * K + N * r) * _BYTES[case["w"]] + 2 * len(ids) * N * _BYTES[case["y"]],
            "flops": 2 * some * r * (S * K + N)}
  _, heads, kv, hd, _ = MODELS[case["model"]]
  row = {"fp32": 4 * hd, "bf16": 2 * hd, "bfp8": hd + hd // 16, "bfp4": hd // 2 + hd // 16}[case["kv"]]
  lens, before, _, _ = _shape(case)
  T = sum(lens)
  if case["kind"] == "append":
    # (each head's row read; q, keys and values written; a place's cos and sin read once)
    n = T * ((heads + 2 * kv) * hd * _BYTES[case["x"]] + heads * hd * _BYTES[case["q"]] + 2 * kv * row + 8 * hd)
    return {"bytes": n, "flops": T * hd * (heads + kv) * (7 if case["norm"] else 3)}
  rows = sum(a + b for a, b in zip(lens, before) if a)
  pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(lens, before))
  return {"bytes": 2 * kv * row * rows + T * heads * hd * (_BYTES[case["q"]] + _BYTES[case["o"]]), "flops": 4 * hd * heads * pairs}


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


def _stands(y):
  """What bfp8 keeps of y [rows][hd]: its bf16 value in whole steps of the run's largest's, halves up, at most 127."""
  v = y.to(torch.bfloat16).double().view(y.shape[0], -1, 16)
  top = torch.frexp(v.abs().amax(2, keepdim=True)).exponent  # (2^(top - 1) <= the largest < 2^top)
  step = torch.ldexp(torch.ones_like(v), top - 7)
  return ((v.abs() / step + 0.5).floor().clamp(max=127) * step * v.sign()).view(y.shape)


def _where(pages, page, n):
  """The cache rows of a sequence's places 0 .. n - 1."""
  return (torch.tensor(pages, dtype=torch.int64, device=DEV)[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)[:n]


def exact(case, seed):
  st = prepare(case, seed)
  if case["kind"] == "lora":
    _, cols, ids = _lora_shape(case)
    r, y, given = st["rank"], st["base"].double(), torch.tensor(ids, device=DEV)
    for i in sorted({i for i in ids if i >= 0}):
      rows = (given == i).nonzero()[:, 0]
      u = st["x"][rows].double() @ st["a"][i].double().T.contiguous()
      at = 0
      for j, c in enumerate(cols):
        y[rows, at:at + c] += st["scale"][i].double() * (u[:, j * r:(j + 1) * r] @ st["b"][i, at:at + c].double().T.contiguous())
        at += c
    return y
  _, heads, kv, hd, _ = MODELS[case["model"]]
  lens, before, own_pages, _ = _shape(case)
  cache, page, at = _exact_cache(case, st, 2 * kv, hd), case["page"], 0
  out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
  if case["kind"] == "append":
    for a, b, pages in zip(lens, before, own_pages):
      if not a: continue
      x = st["x"][at:at + a].double().view(a, heads + 2 * kv, hd)
      to = _where(pages, page, a + b)[b:]
      c, s = st["cos"][b:b + a, :hd // 2].double(), st["sin"][b:b + a, :hd // 2].double()
      for h in range(heads + 2 * kv):
        y = x[:, h]
        if h < heads + kv:
          if case["norm"]: y = y / torch.sqrt((y ** 2).sum(1, keepdim=True) / hd + EPS) * (st["q_norm"] if h < heads else st["k_norm"]).double()
          one, two = y[:, :hd // 2], y[:, hd // 2:]
          y = torch.cat([one * c - two * s, two * c + one * s], 1)
        if h < heads: out[at:at + a, h * hd:(h + 1) * hd] = y
        else: cache[h - heads, to] = y if case["kv"] in DTYPE else _stands(y)
      at += a
    return out, cache
  rep = heads // kv
  for a, b, pages in zip(lens, before, own_pages):
    if not a: continue
    where, hidden = _where(pages, page, a + b), torch.arange(a + b, device=DEV)[None] > b + torch.arange(a, device=DEV)[:, None]
    for g in range(kv):
      k, v = cache[g][where], cache[kv + g][where]
      for h in range(g * rep, (g + 1) * rep):
        s = (st["q"][at:at + a, h * hd:(h + 1) * hd].double() @ k.T.contiguous()) / math.sqrt(hd)
        out[at:at + a, h * hd:(h + 1) * hd] = torch.softmax(s.masked_fill(hidden, -math.inf), 1) @ v
    at += a
  return out
