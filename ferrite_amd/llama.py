"""A Llama decoder on MI355X: models/llama.py's layer structure (layer -> attention / mlp -> mm, models/llama.py:95-146,
266-269, 459-480) run as the library's fused kernels, a step replayable as one HIP graph (tensor.jit's place,
ferrite/tensor.py:775-810).

A decode step of `batch` rows (one token of each of `batch` sequences, or a prompt's tokens at consecutive places)
is, per block:
  qkv     fh_gemv_bfp  RMSNorm prologue, RoPE on q's and k's heads, k and v put into the cache at each row's place
  attend  fh_attention_decode over the rows each place reaches
  o       fh_gemv_bfp  + the residual (x += o), with x's sums of squares for the next norm
  gate_up fh_gemv_bfp  RMSNorm prologue, silu(gate) * up
  down    fh_gemv_bfp  + the residual
then the final norm and the output layer (fp32 logits) and each row's argmax. Activations stay fp32 between
kernels; weights are block floats (precision's formats); the KV cache is bf16 or fp32.

A prompt (prefill: T tokens at consecutive places of one sequence, models/llama.py:498-504) runs on the matrix cores,
the residual stream fp32 and each GEMM's input bf16 (as ferrite's chip feeds its matrix unit), per block:
  norm    fh_rms_rows  x -> bf16 rows
  qkv     fh_gemm_bfp  RoPE on q's and k's heads, k and v put into the cache at each row's place
  attend  fh_attention_prefill, causal over the sequence's rows (bf16 out)
  o       fh_gemm_bfp  + the residual
  norm    fh_rms_rows
  gate_up fh_gemm_bfp  silu(gate) * up (bf16 out)
  down    fh_gemm_bfp  + the residual, with x's sums of squares
then the final norm and the output layer for the last row only (fh_gemv_bfp), and its argmax.

Many prompts go in together (prefill_batch): their rows packed one after another through the same matmuls, the attention
fh_attention_prefill_packed. A batch whose sequences begin alike keeps that prefix once (share_prefix): its rows' attention is
fh_attention_decode_shared, their own slots hold what follows the prefix.

A service whose sequences' lengths are anybody's guess keeps them in pages of the same cache, and its requests may bring low-rank adapters
(step_pages; page_step for a decode step replayed as one HIP graph). qkv is then a plain product, which fh_lora adds each row's adapter to;
fh_rope_append_paged turns it and puts k and v into the rows' pages, and the attention is fh_attention_paged. o, gate_up and down take
fh_lora behind their products the same way.
"""
import math
from types import SimpleNamespace
import numpy as np
import torch
from ferrite_amd import lib, ops


PUT_MAX = 4096  # a prompt's tokens that go to the GPU as launches' arguments (5 launches); more by copies


def model(**c):
  """A config: dim, heads, kv, layers, eps, theta, vocab, ffn, places (RoPE rows), head_dim, rope (Llama 3's scaling),
  tied (output layer = embedding), centered (RMSNorm by 1 + w), as models/llama.py:541-543 keeps them."""
  d = dict(head_dim=None, rope=None, centered=False, tied=False, places=4096, k=0, experts=0, norm_topk=True)
  return SimpleNamespace(**(d | c))


def head(c): return c.head_dim or c.dim // c.heads


def precision(c, mode="bfp8"):
  """Each matrix's format (models/llama.py:54-76): bfp8 (all), bfp4 (the MLP's gate and up in bfp4), experts (every MLP
  matrix in bfp4), the rest bfp8. (Fidelity phases are the chip's: products here are exact.)"""
  four = {"bfp4": ("gate_up",), "tt": ("gate_up",), "experts": ("gate_up", "down")}.get(mode, ())
  if mode not in ("bfp8", "bfp4", "tt", "experts"): raise ValueError(f"precision: {mode} (the GPU path reads block floats)")
  p = {(op, l): ("bfp4" if op in four else "bfp8") for l in range(c.layers) for op in ("qkv", "o", "gate_up", "down")}
  if mode == "tt" and (c.layers, c.dim) == (32, 4096): p["gate_up", 31] = "bfp8"
  p["head", None] = "bfp8"
  return p


def frequencies(c):
  """RoPE's inverse frequencies in fp32, Llama 3's scaling if c.rope says llama3 (models/llama.py:333-344)."""
  hd = head(c)
  inv = 1 / c.theta ** (np.arange(0, hd, 2, dtype=np.float32) / hd)
  r = c.rope
  if r and r.get("rope_type") == "llama3":
    old, wavelen = r["original_max_position_embeddings"], 2 * math.pi / inv
    scaled = np.where(wavelen > old / r["low_freq_factor"], inv / r["factor"], inv)
    smooth = (old / wavelen - r["low_freq_factor"]) / (r["high_freq_factor"] - r["low_freq_factor"])
    between = (wavelen >= old / r["high_freq_factor"]) & (wavelen <= old / r["low_freq_factor"])
    inv = np.where(between, (1 - smooth) * scaled / r["factor"] + smooth * scaled, scaled).astype(np.float32)
  return inv


def rotary_tables(c, n):
  """One head's cos and sin for places 0..n-1, (n, head_dim) fp32 holding bf16 values: fp32 angles rounded to bf16,
  each half the same (models/llama.py:354-368; the kernel applies them to every q and k head)."""
  angles = np.arange(n, dtype=np.float32)[:, None] * frequencies(c)[None]
  def bf16(a):
    b = np.asarray(a, np.float32).view(np.uint32).astype(np.uint64)
    return (((b + 0x7FFF + (b >> 16 & 1)) >> 16 & 0xFFFF).astype(np.uint32) << 16).view(np.float32)
  return bf16(np.concatenate([np.cos(angles)] * 2, 1)), bf16(np.concatenate([np.sin(angles)] * 2, 1))


class Decoder:
  """The model's weights on the GPU (block floats by precision), its KV cache, and the buffers of a step of `batch`
  rows. weights(name, shape) gives each weight as a torch fp32 (or bf16) tensor on the GPU, named as models/llama.py's
  fuse leaves them: layers.{l}.input_layernorm, .post_attention_layernorm, .qkv_proj, .o_proj, .gate_up_proj,
  .down_proj (x @ w), norm, embed, embed.T (the output layer; the embedding's transpose when tied)."""

  def __init__(self, c, weights, mode="bfp8", kv="bf16", batch=1, context=256, device="cuda", slots=1, mfma_from=3,
               share=None):
    """mfma_from: the batch from which a step's matmuls run on the matrix cores (fh_gemm_bfp, bf16 rows) rather than
    the exact-product GEMV (None: never); 3 by default, where the two meet on MI355X (an 8B step: 3.0 ms either way at
    3 rows, 3.06 against 3.42 at 4, 3.44 against 6.49 at 8). share: another Decoder of the same model whose weights this one uses."""
    self.c, self.mode, self.batch, self.context, self.device = c, mode, batch, context, torch.device(device)
    self.prec = precision(c, mode)
    hd = head(c)
    self.hd, self.qkv_cols = hd, (c.heads + 2 * c.kv) * hd
    self.mm = ops.gemm if mfma_from is not None and batch >= mfma_from else ops.gemv
    if share is not None:
      self.layers, self.norm, self.embed, self.head, self.cos, self.sin = share.layers, share.norm, share.embed, share.head, share.cos, share.sin
    else:
      self._load(weights)
    self._buffers(kv, batch, context, slots)

  def _load(self, weights):
    """weights: weights(name, shape) giving x @ W's layout (numpy_weights, random_weights), or a checkpoint.Checkpoint,
    whose matrices are packed straight from its rows (fused and transposed in the packing)."""
    c, hd = self.c, self.hd
    ck = weights if hasattr(weights, "pack") else None
    f32 = lambda t: t.to(self.device, torch.float32).contiguous()

    def mat(name, K, N, fmt):
      bw = ck.pack(name, fmt) if ck is not None else ops.pack(weights(name, (K, N)).to(self.device), fmt)
      if (bw.K, bw.N) != (K, N): raise ValueError(f"{name}: {bw.K}x{bw.N}, the model says {K}x{N}")
      return bw

    def vec(name):
      return ck.vector(name) if ck is not None else f32(weights(name, (1, c.dim))).reshape(-1)

    self.layers = []
    for l in range(c.layers):
      pre = f"layers.{l}."
      L = SimpleNamespace()
      L.norm1, L.norm2 = vec(pre + "input_layernorm"), vec(pre + "post_attention_layernorm")
      L.qkv = mat(pre + "qkv_proj", c.dim, self.qkv_cols, self.prec["qkv", l])
      L.o = mat(pre + "o_proj", c.heads * hd, c.dim, self.prec["o", l])
      L.gate_up = mat(pre + "gate_up_proj", c.dim, 2 * c.ffn, self.prec["gate_up", l])
      L.down = mat(pre + "down_proj", c.ffn, c.dim, self.prec["down", l])
      self.layers.append(L)
    self.norm = vec("norm")
    # the embedding in bf16 (a row read per token); the output layer its own matrix, or the embedding's rows packed
    # as its transpose (tied)
    self.embed = ck.table() if ck is not None else weights("embed", (c.vocab, c.dim)).to(self.device, torch.bfloat16).contiguous()
    if ck is not None: self.head = mat("embed.T", c.dim, c.vocab, self.prec["head", None])
    elif c.tied: self.head = ops.pack_parts([self.embed], self.prec["head", None])
    else: self.head = mat("embed.T", c.dim, c.vocab, self.prec["head", None])
    cos, sin = rotary_tables(c, c.places)
    self.cos, self.sin = torch.from_numpy(cos).to(self.device), torch.from_numpy(sin).to(self.device)

  def _buffers(self, kv, batch, context, slots):
    c, hd = self.c, self.hd
    # the KV cache: a block's keys' heads then values', `slots` sequences' rows side by side (models/llama.py:506-514)
    self.slots = slots or 1
    self.part = context  # rows a sequence
    # (bfp8 / bfp4: a block-float cache, each run of 16 of a row rounded as the qkv epilogue puts it; llama.py:127-128)
    if kv not in ("fp32", "bf16", "bfp8", "bfp4"): raise ValueError(f"kv cache: fp32, bf16, bfp8 or bfp4, not {kv}")
    self.kv = kv
    self.cache = [ops.kv_cache(2 * c.kv, self.slots * context, hd, kv, self.device) for _ in range(c.layers)]
    # a step's buffers, fixed so a step replays as a graph
    B = batch
    z = lambda *s: torch.zeros(*s, dtype=torch.float32, device=self.device)
    # each row's token, place, its sequence's first cache row and the cache row of its token: one buffer, so that a
    # step's values from the host go in by one launch
    self._int = torch.zeros(4, B, dtype=torch.int32, device=self.device)
    self.ids, self.places, self.first, self.rows = self._int
    self.x, self.ssq = z(B, c.dim), z(B, c.dim // 16)
    self.q, self.att = z(B, c.heads * hd), z(B, c.heads * hd)
    self.h = z(B, c.ffn)
    # the matrix cores' bf16 rows: each residual epilogue's copy, SwiGLU's output, attention's output for o; in tiles of
    # 16 rows (FH_BF16_T16) up to 64 rows, which the matrix-core kernel for a few rows loads a whole line at a time. That
    # kernel takes K a multiple of 64 only: a model with any matmul's K (dim, heads head_dim, ffn) off that keeps plain
    # bf16 rows, which the tiled GEMM takes at any K
    tiled = B <= 64 and all(k % 64 == 0 for k in (c.dim, c.heads * hd, c.ffn))
    rows16 = ops.tiles16 if tiled else (lambda r, n, d: torch.zeros(r, n, dtype=torch.bfloat16, device=d))
    self.xn = rows16(B, c.dim, self.device)
    self.hb = rows16(B, c.ffn, self.device)
    self.attb = rows16(B, c.heads * hd, self.device)
    self.logits = z(B, c.vocab)
    self.picks = torch.zeros(B, dtype=torch.int32, device=self.device)
    self.parts = torch.zeros(B, c.vocab // 16, dtype=torch.int64, device=self.device)  # each run of 16 logits' best
    self.ws = ops.attention_workspace(B, c.heads, hd, context, self.device)
    self.graph = None
    # the shared prefix (share_prefix): its slot, its places, each row's of them, the same on the GPU; none at first
    self.prefix_slot, self.prefix_len, self.shared_host = None, 0, np.zeros(B, np.int32)
    self.prefix_row, self.shared = (torch.zeros(n, dtype=torch.int32, device=self.device) for n in (1, B))
    self.top = 0  # the largest place of the rows set (set_rows), which advance raises,
    self.top_own = 0  # and the largest behind the prefix: the row of its slot
    self.placed = True  # (False from a change of the sharing until the rows are set again)
    self.behind = np.full(self.slots, -1, np.int64)  # the prefix's places before each slot's rows, where known (_follow)
    self.sharing = False  # (a prefix was shared at some time)

  def weight_bytes(self):
    """Bytes of the weights one decode step reads: every matrix, a row of the embedding, the norms."""
    n = sum(w.nbytes for L in self.layers for w in (L.qkv, L.o, L.gate_up, L.down)) + self.head.nbytes
    return n + self.c.dim * 2 + (2 * self.c.layers + 1) * self.c.dim * 4

  def set_rows(self, places, slots=None):
    """Each row's place, and the cache rows: slot s's sequence keeps rows s * context .. (models/llama.py:429-452), from the
    first place behind the prefix on where the row shares one (share_prefix)."""
    self._put(places=places, slots=slots)

  def _follow(self, what, slots, shared, own):
    """Slots whose rows follow the first shared[i] places of the prefix, written from row own[i] on: noted where a slot begins anew
    (row 0), and refused where it holds rows known to follow another number of places, which would be read as what they are not."""
    slots, shared, own = np.asarray(slots), np.asarray(shared), np.asarray(own)
    held = self.behind[slots]
    bad = (own > 0) & (held != -1) & (held != shared)
    if bad.any():
      i = int(bad.argmax())
      raise ValueError(f"{what}: slot {slots[i]} holds what follows {held[i]} places of a prefix, not {shared[i]}")
    anew = own == 0
    self.behind[slots[anew]] = shared[anew]

  def share_prefix(self, slot=None, length=0, rows=None):
    """The first `length` places of slot `slot` (a prompt prefilled there) become the prefix of the batch's sequences: row b
    shares the first rows[b] of them (all of them by default), kept once and read for many rows at a time, and its own slot holds
    its places from rows[b] on. A sequence may then have rows[b] + context places. The prefix's slot is not a row's while one
    shares it, and a slot filled behind one number of places is refused to a row that shares another. share_prefix() ends it. The
    rows are set again afterwards (set_rows, step's places); a step captured before is captured again where the length changes."""
    if slot is None:
      length, rows = 0, np.zeros(self.batch, np.int32)
    else:
      if not 0 <= slot < self.slots: raise ValueError(f"share_prefix: slot {slot} outside 0..{self.slots - 1}")
      if not 1 <= length <= min(self.context, self.c.places): raise ValueError(f"share_prefix: {length} places of a slot of {self.context}")
      rows = np.full(self.batch, length, np.int32) if rows is None else np.array(rows, np.int32)  # (a copy: the caller may write to its own)
      if rows.shape != (self.batch,) or (rows < 0).any() or (rows > length).any(): raise ValueError(f"share_prefix: {self.batch} rows' counts in 0..{length}")
      if self.behind[slot] > 0: raise ValueError(f"share_prefix: slot {slot} holds what follows {self.behind[slot]} places of a prefix, not a prompt from its first place on")
      ops.attention_heads_ok(self.c.heads, self.c.kv, self.hd)
      self.sharing = True
    # (the captured step reads the slot's first row and the counts when it runs; another length is another launch)
    if (slot is None) != (self.prefix_slot is None) or int(length) != self.prefix_len:
      if self.graph is not None: torch.cuda.synchronize(self.device)  # (a replay may be running)
      self.ws_shared = ops.attention_shared_workspace(self.batch, self.c.heads, self.c.kv, self.hd, length, self.context, self.device) if slot is not None else None
      self.graph = None  # (the step is captured again)
    self.prefix_slot, self.prefix_len, self.shared_host = slot, int(length), rows
    ops.put_i32(rows, self.shared)
    ops.put_i32([(slot or 0) * self.part], self.prefix_row)
    self.placed = False

  def _attend(self, l, out):
    """A step's attention over block l's cache."""
    c = self.c
    if self.prefix_slot is None:
      ops.attention_decode(self.q, self.cache[l], c.heads, c.kv, self.hd, self.places, self.first, self.context, self.ws, o=out)
    else:
      ops.attention_decode_shared(self.q, self.cache[l], c.heads, c.kv, self.hd, self.places, self.first, self.prefix_row, self.shared,
                                  self.prefix_len, self.context, workspace=self.ws_shared, o=out)

  def _put(self, ids=None, places=None, slots=None):
    """The rows' tokens, and their places and slots where places is given: what the host holds by one launch whose
    arguments they are (ops.put_i32), tensors on the GPU by copies on the stream."""
    if ids is not None:
      ids = torch.as_tensor(ids, dtype=torch.int32)
      if places is None or ids.is_cuda or ids.shape != (self.batch,):
        if ids.is_cuda or ids.shape != (self.batch,): self.ids.copy_(ids)
        else: ops.put_i32(ids.numpy(), self.ids)
        ids = None
    if places is None: return
    places = torch.as_tensor(places, dtype=torch.int32)
    slots = torch.zeros_like(places) if slots is None else torch.as_tensor(slots, dtype=torch.int32)
    if places.shape != (self.batch,) or slots.shape != (self.batch,): raise ValueError(f"set_rows: {self.batch} places and slots")
    host = not (places.is_cuda or slots.is_cuda)
    p, s = (places.numpy(), slots.numpy()) if host else (places, slots)
    sh = self.shared_host if host else self.shared
    if not host: p, s = p.to(self.device), s.to(self.device)
    if (p < sh).any() or (p - sh >= self.context).any() or (p >= self.c.places).any(): raise ValueError("a place inside the shared prefix, or past the cache or RoPE's tables")
    if (s < 0).any() or (s >= self.slots).any(): raise ValueError(f"a slot outside 0..{self.slots - 1}")
    if self.prefix_slot is not None and (s == self.prefix_slot).any(): raise ValueError(f"slot {self.prefix_slot} holds the shared prefix")
    if self.sharing:
      host_of = (lambda t: t) if host else (lambda t: t.cpu().numpy())
      self._follow("set_rows", host_of(s), self.shared_host, host_of(p - sh))
    self.top, self.top_own = int(p.max()), int((p - sh).max())  # (kept on the host for advance's check)
    self.placed = True
    if host:
      first = s * np.int32(self.part)
      v = [p, first, first + p - sh]
      ops.put_i32(np.concatenate(v if ids is None else [ids.numpy(), *v]), self._int[1 if ids is None else 0:])
      return
    if ids is not None: ops.put_i32(ids.numpy(), self.ids)
    self.places.copy_(p)
    self.first.copy_(s * self.part)
    self.rows.copy_(s * self.part + p - sh)

  def _cache(self, l):
    data, dtype, length = ops.cache_fields(self.cache[l])
    return dict(cache=data, cache_dtype=dtype, cache_len=length)

  def _step(self):
    if self.mm is ops.gemm: return self._step_rows()
    c, B, hd = self.c, self.batch, self.hd
    ops.embed_rows(self.embed, self.ids, self.x, self.ssq)
    for l, L in enumerate(self.layers):
      ep = ops.epilogue(lib.EP_ROPE_KV, norm_w=L.norm1, ssq_in=self.ssq, eps=c.eps, centered=int(c.centered),
                        heads=c.heads, kv_heads=c.kv, head_dim=hd, cos_tab=self.cos, sin_tab=self.sin, rope_rows=self.cos.shape[0],
                        places=self.places, cache_rows=self.rows, **self._cache(l))
      ops.gemv(self.x, L.qkv, ep, out=self.q)
      self._attend(l, self.att)
      ep = ops.epilogue(lib.EP_RESIDUAL, residual=self.x, ssq_out=self.ssq)
      ops.gemv(self.att, L.o, ep, out=self.x)
      ep = ops.epilogue(lib.EP_SILU_GATE, norm_w=L.norm2, ssq_in=self.ssq, eps=c.eps, centered=int(c.centered), split=c.ffn)
      ops.gemv(self.x, L.gate_up, ep, out=self.h)
      ep = ops.epilogue(lib.EP_RESIDUAL, residual=self.x, ssq_out=self.ssq)
      ops.gemv(self.h, L.down, ep, out=self.x)
    ep = ops.epilogue(lib.EP_STORE, norm_w=self.norm, ssq_in=self.ssq, eps=c.eps, centered=int(c.centered), argmax_parts=self.parts)
    ops.gemv(self.x, self.head, ep, out=self.logits)
    ops.argmax_parts(self.parts, self.picks)

  def _norm_weights(self):
    """Each RMSNorm's multiplier (its weight, + 1 where centered) in the order a step meets them: block l's norm1,
    norm2, ..., then the final norm."""
    if getattr(self, "_nw", None) is None:
      c = self.c
      ws = [w for L in self.layers for w in (L.norm1, L.norm2)] + [self.norm]
      self._nw = [w + 1 if c.centered else w for w in ws]
    return self._nw

  def _step_rows(self):
    """A step of many rows on the matrix cores. The residual stream stays fp32; each residual epilogue also writes
    its rows times the next RMSNorm's weight in bf16 (copy_bf16, copy_w) with their sums of squares, and the next
    matmul takes those rows scaled by 1/rms (ssq_in alone): the products are its RMSNorm prologue's, bf16(x w), with
    no normalising pass (the first block's norm a kernel of its own). SwiGLU's output bf16."""
    c, B, hd = self.c, self.batch, self.hd
    nw = self._norm_weights()
    ops.embed_rows(self.embed, self.ids, self.x, self.ssq)
    rs = dict(ssq_in=self.ssq, eps=c.eps)  # rows that hold x w: 1/rms only
    for l, L in enumerate(self.layers):
      rope = dict(heads=c.heads, kv_heads=c.kv, head_dim=hd, cos_tab=self.cos, sin_tab=self.sin, rope_rows=self.cos.shape[0], places=self.places,
                  cache_rows=self.rows, **self._cache(l))
      if l == 0:
        ops.rms_rows(self.x, L.norm1, c.eps, c.centered, out=self.xn)
        ops.gemm(self.xn, L.qkv, ops.epilogue(lib.EP_ROPE_KV, **rope), out=self.q)
      else:
        ops.gemm(self.xn, L.qkv, ops.epilogue(lib.EP_ROPE_KV, **rs, **rope), out=self.q)
      self._attend(l, self.attb)
      ops.gemm(self.attb, L.o, ops.epilogue(lib.EP_RESIDUAL, residual=self.x, ssq_out=self.ssq, copy_bf16=self.xn,
                                           copy_w=nw[2 * l + 1]), out=self.x)
      ops.gemm(self.xn, L.gate_up, ops.epilogue(lib.EP_SILU_GATE, split=c.ffn, **rs), out=self.hb)
      ops.gemm(self.hb, L.down, ops.epilogue(lib.EP_RESIDUAL, residual=self.x, ssq_out=self.ssq, copy_bf16=self.xn,
                                             copy_w=nw[2 * l + 2]), out=self.x)
    ops.gemm(self.xn, self.head, ops.epilogue(lib.EP_STORE, argmax_parts=self.parts, **rs), out=self.logits)
    ops.argmax_parts(self.parts, self.picks)

  def _prefill_buffers(self, T):
    c, hd, dev = self.c, self.hd, self.device
    P = getattr(self, "_pre", None)
    if P is None or P.T < T:
      z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=dev)
      P = SimpleNamespace(T=T, ids=z(T, dtype=torch.int32), places=z(T, dtype=torch.int32), rows=z(T, dtype=torch.int32),
                          x=z(T, c.dim), ssq=z(T, c.dim // 16), xn=z(T, c.dim, dtype=torch.bfloat16), q=z(T, c.heads * hd),
                          att=z(T, c.heads * hd, dtype=torch.bfloat16), h=z(T, c.ffn, dtype=torch.bfloat16),
                          logits=z(1, c.vocab), parts=z(1, c.vocab // 16, dtype=torch.int64), pick=z(1, dtype=torch.int32))
      self._pre = P
    return P

  def prefill(self, ids, slot=0, p0=0, chunk=None):
    """A prompt's tokens at places p0 .. p0 + len(ids) - 1 of sequence `slot`, on the matrix cores (in chunks of
    `chunk` tokens, as models/llama.py:498-504 prefills): their keys and values go into the cache; returns the last
    token's logits ([1][vocab] fp32) and its greedy pick ([1] int32). Each call repeats its bits, but chunks give the
    whole prompt's values within the rounding of fp32 sums: the order in which a matmul adds K and attention the keys
    follows the rows of a call."""
    ids = [int(i) for i in ids]
    T = len(ids)
    if T < 1 or p0 < 0 or p0 + T > min(self.context, self.c.places): raise ValueError("prefill: the prompt's places past the cache or RoPE's tables")
    if not 0 <= slot < self.slots: raise ValueError(f"prefill: slot {slot} outside 0..{self.slots - 1}")
    if self.prefix_slot not in (None, slot): raise ValueError("prefill: sequences behind a shared prefix go through prefill_batch")
    self._follow("prefill", [slot], [0], [p0])
    chunk = chunk or T
    for a in range(0, T, chunk):
      out = self._prefill_chunk(ids[a:a + chunk], slot, p0 + a)
    return out

  def _prefill_chunk(self, ids, slot, p0):
    c, hd = self.c, self.hd
    T = len(ids)
    P = self._prefill_buffers(T)
    ids_t, places, rows = P.ids[:T], P.places[:T], P.rows[:T]
    x, ssq, xn, q, att, h = P.x[:T], P.ssq[:T], P.xn[:T], P.q[:T], P.att[:T], P.h[:T]
    at = np.arange(p0, p0 + T, dtype=np.int32)
    if T <= PUT_MAX:
      for v, out in ((ids, ids_t), (at, places), (at + np.int32(slot * self.part), rows)): ops.put_i32(v, out)
    else:
      for v, out in ((ids, ids_t), (at, places), (at + np.int32(slot * self.part), rows)): out.copy_(torch.as_tensor(v, dtype=torch.int32))
    ops.embed_rows(self.embed, ids_t, x, ssq)
    # (each RMSNorm a pass of its own here: at 2048 rows the tiled kernel's per-tile sums of the rows' squares cost
    # more than fh_rms_rows; the batched decode takes the residual epilogues' scaled copies instead)
    for l, L in enumerate(self.layers):
      ops.rms_rows(x, L.norm1, c.eps, c.centered, out=xn)
      ep = ops.epilogue(lib.EP_ROPE_KV, heads=c.heads, kv_heads=c.kv, head_dim=hd, cos_tab=self.cos, sin_tab=self.sin, rope_rows=self.cos.shape[0],
                        places=places, cache_rows=rows, **self._cache(l))
      ops.gemm(xn, L.qkv, ep, out=q)
      ops.attention_prefill(q, self.cache[l], c.heads, c.kv, hd, p0, slot * self.part, o=att)
      ops.gemm(att, L.o, ops.epilogue(lib.EP_RESIDUAL, residual=x), out=x)
      ops.rms_rows(x, L.norm2, c.eps, c.centered, out=xn)
      ops.gemm(xn, L.gate_up, ops.epilogue(lib.EP_SILU_GATE, split=c.ffn), out=h)
      ops.gemm(h, L.down, ops.epilogue(lib.EP_RESIDUAL, residual=x, ssq_out=ssq), out=x)
    ep = ops.epilogue(lib.EP_STORE, norm_w=self.norm, ssq_in=ssq[T - 1:], eps=c.eps, centered=int(c.centered), argmax_parts=P.parts)
    ops.gemv(x[T - 1:], self.head, ep, out=P.logits)
    ops.argmax_parts(P.parts, P.pick)
    return P.logits, P.pick

  def prefill_batch(self, prompts, slots=None, p0=None, shared=None):
    """Prompts of many sequences at once, on the matrix cores: prompt i's tokens at places p0[i], p0[i] + 1, ... of slot
    slots[i] (slot i by default), each slot once; the first shared[i] places are the prefix's (share_prefix; by default all of them,
    none without one) and p0 begins behind them by default. The row that steps a slot later shares as many (share_prefix's rows;
    set_rows refuses another count). Their keys and values go into the cache; returns each prompt's last token's logits
    ([n][vocab] fp32) and greedy picks ([n] int32). The rows of all prompts go through the matmuls together, so a prompt's
    logits have prefill's values within the rounding of bf16 rows and fp32 sums."""
    c, hd, dev = self.c, self.hd, self.device
    n = len(prompts)
    ops.attention_heads_ok(c.heads, c.kv, hd)  # (before any block's keys are put)
    if n < 1: raise ValueError("prefill_batch: no prompt")
    lens = np.array([len(p) for p in prompts], np.int64)
    slots = np.arange(n) if slots is None else np.asarray(slots, np.int64)
    sh = np.full(n, self.prefix_len, np.int64) if shared is None else np.asarray(shared, np.int64)
    p0 = sh if p0 is None else np.asarray(p0, np.int64)
    if not slots.shape == sh.shape == p0.shape == (n,): raise ValueError(f"prefill_batch: {n} slots, p0 and shared")
    if (lens < 1).any(): raise ValueError("prefill_batch: an empty prompt")
    if (slots < 0).any() or (slots >= self.slots).any() or len(set(slots.tolist())) != n: raise ValueError(f"prefill_batch: each slot once, in 0..{self.slots - 1}")
    if (sh < 0).any() or (sh > self.prefix_len).any(): raise ValueError(f"prefill_batch: shared in 0..{self.prefix_len}")
    if self.prefix_slot is not None and (slots == self.prefix_slot).any(): raise ValueError(f"prefill_batch: slot {self.prefix_slot} holds the shared prefix")
    if (p0 < sh).any() or (p0 - sh + lens > self.context).any() or (p0 + lens > c.places).any():
      raise ValueError("prefill_batch: a prompt's places inside the shared prefix, or past the cache or RoPE's tables")
    self._follow("prefill_batch", slots, sh, p0 - sh)
    T, starts = int(lens.sum()), np.concatenate([[0], np.cumsum(lens)])
    P = self._prefill_buffers(T)
    of = np.repeat(np.arange(n), lens)  # each row's prompt
    places = np.arange(T) - starts[of] + p0[of]
    rows = slots[of] * self.part + places - sh[of]
    ids = np.concatenate([np.asarray(p, np.int64) for p in prompts])
    ints = np.concatenate([ids, places, rows, starts, p0, slots * self.part, sh, starts[1:] - 1]).astype(np.int32)
    held = torch.empty(ints.size, dtype=torch.int32, device=dev)
    if ints.size <= PUT_MAX: ops.put_i32(ints, held)
    else: held.copy_(torch.from_numpy(ints))
    ids_t, places_t, rows_t, starts_t, p0_t, first_t, sh_t, last_t = held.split([T, T, T, n + 1, n, n, n, n])
    prefix = dict(prefix_row=self.prefix_row, shared=sh_t) if sh.any() else {}
    most = int((p0 + lens).max())
    ws = ops.attention_packed_workspace(T, n, c.heads, c.kv, hd, most, dev)
    x, ssq, xn, q, att, h = P.x[:T], P.ssq[:T], P.xn[:T], P.q[:T], P.att[:T], P.h[:T]
    ops.embed_rows(self.embed, ids_t, x, ssq)
    for l, L in enumerate(self.layers):
      ops.rms_rows(x, L.norm1, c.eps, c.centered, out=xn)
      ep = ops.epilogue(lib.EP_ROPE_KV, heads=c.heads, kv_heads=c.kv, head_dim=hd, cos_tab=self.cos, sin_tab=self.sin, rope_rows=self.cos.shape[0],
                        places=places_t, cache_rows=rows_t, **self._cache(l))
      ops.gemm(xn, L.qkv, ep, out=q)
      ops.attention_prefill_packed(q, self.cache[l], c.heads, c.kv, hd, starts_t, p0_t, first_t, most, workspace=ws, o=att, **prefix)
      ops.gemm(att, L.o, ops.epilogue(lib.EP_RESIDUAL, residual=x), out=x)
      ops.rms_rows(x, L.norm2, c.eps, c.centered, out=xn)
      ops.gemm(xn, L.gate_up, ops.epilogue(lib.EP_SILU_GATE, split=c.ffn), out=h)
      ops.gemm(h, L.down, ops.epilogue(lib.EP_RESIDUAL, residual=x), out=x)
    return self._last_rows(x, last_t, n)

  def _page_layout(self, what, places, lens, tables, page):
    """The tables [n][pages] of sequences whose rows are at places[i] .. places[i] + lens[i] - 1, checked: pages that the cache has (-1
    behind those that a sequence needs), and no page that rows are put into another's."""
    pages = self.slots * self.part // page if page > 0 else 0
    if page < 16 or page & (page - 1) or self.slots * self.part % page: raise ValueError(f"{what}: pages of 16, 32, 64, ... rows of a cache of {self.slots * self.part}")
    n = len(lens)
    if len(tables) != n or places.shape != (n,): raise ValueError(f"{what}: {n} places and tables")
    if (places < 0).any() or (places + lens > self.c.places).any(): raise ValueError(f"{what}: a place outside RoPE's tables")
    need = -(-(places + lens) // page)
    out = np.full((n, max(int(need.max()), max(len(t) for t in tables))), -1, np.int64)
    for i, t in enumerate(tables):
      if len(t) < need[i]: raise ValueError(f"{what}: sequence {i} needs {need[i]} pages, not {len(t)}")
      out[i, :len(t)] = t
    col = np.arange(out.shape[1])[None]
    used = col < need[:, None]
    if ((out[used] < 0) | (out[used] >= pages)).any(): raise ValueError(f"{what}: a page outside 0..{pages - 1}")
    written = out[used & (col >= (places // page)[:, None])]
    if (np.bincount(out[used], minlength=pages)[written] > 1).any(): raise ValueError(f"{what}: a page that rows are put into is another's too")
    return out

  def _page_rows(self, P, T, n, ids, starts, p0, last, of, tables, page, most, ws, adapters):
    """The model over T packed rows of n sequences whose keys and values lie in pages: each sequence's last row's logits and pick. of:
    each row's adapter, where there are any."""
    c, hd = self.c, self.hd
    x, ssq, xn, q, att, h = P.x[:T], P.ssq[:T], P.xn[:T], P.q[:T], P.att[:T], P.h[:T]
    lora_ws = P.lora_ws if adapters else None
    ops.embed_rows(self.embed, ids, x, ssq)
    for l, L in enumerate(self.layers):
      ad = adapters[l] if adapters else {}
      ops.rms_rows(x, L.norm1, c.eps, c.centered, out=xn)
      qkv = ops.gemm(xn, L.qkv, out=P.qkv[:T])
      if "qkv" in ad: ops.lora(xn, ad["qkv"], of, residual=qkv, out=qkv, workspace=lora_ws)
      ops.rope_append_paged(qkv, self.cache[l], c.heads, c.kv, hd, self.cos, self.sin, starts, p0, tables, page, q=q)
      ops.attention_paged(q, self.cache[l], c.heads, c.kv, hd, starts, p0, tables, page, most, workspace=ws, o=att)
      ops.gemm(att, L.o, ops.epilogue(lib.EP_RESIDUAL, residual=x), out=x)
      if "o" in ad: ops.lora(att, ad["o"], of, residual=x, out=x, workspace=lora_ws)
      ops.rms_rows(x, L.norm2, c.eps, c.centered, out=xn)
      if "gate_up" in ad:
        gu = ops.gemm(xn, L.gate_up, out=P.gu[:T])
        ops.lora(xn, ad["gate_up"], of, residual=gu, out=gu, workspace=lora_ws)
        ops.silu_gate_rows(gu, c.ffn, h)
      else:
        ops.gemm(xn, L.gate_up, ops.epilogue(lib.EP_SILU_GATE, split=c.ffn), out=h)
      ops.gemm(h, L.down, ops.epilogue(lib.EP_RESIDUAL, residual=x), out=x)
      if "down" in ad: ops.lora(h, ad["down"], of, residual=x, out=x, workspace=lora_ws)
    return self._last_rows(x, last, n)

  def _page_buffers(self, T, adapters):
    c, hd, dev = self.c, self.hd, self.device
    e = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype, device=dev)
    b = torch.bfloat16
    P = SimpleNamespace(T=T, x=e(T, c.dim), ssq=e(T, c.dim // 16), xn=e(T, c.dim, dtype=b), qkv=e(T, self.qkv_cols), q=e(T, c.heads * hd), att=e(T, c.heads * hd, dtype=b), h=e(T, c.ffn, dtype=b))
    if adapters:
      given = [a for ad in adapters for a in ad.values()]
      if any("gate_up" in ad for ad in adapters): P.gu = e(T, 2 * c.ffn)
      P.lora_ws = max((ops.lora_workspace(T, a, dev) for a in given), key=lambda t: t.numel())
    return P

  def _check_adapters(self, what, adapters):
    """The blocks' adapters (None: none), checked, in lists and dicts of their own: what a captured step reads is not the caller's to replace."""
    c, qkv = self.c, (self.c.heads * self.hd, self.c.kv * self.hd, self.c.kv * self.hd)
    shapes = dict(qkv=(c.dim, qkv), o=(c.heads * self.hd, (c.dim,)), gate_up=(c.dim, (c.ffn, c.ffn)), down=(c.ffn, (c.dim,)))
    if adapters is None or not any(adapters): return None
    if len(adapters) != c.layers: raise ValueError(f"{what}: adapters for each of {c.layers} blocks")
    for ad in adapters:
      for name, a in ad.items():
        if name not in shapes or (a.a.shape[2], a.parts) != shapes[name]: raise ValueError(f"{what}: {name}'s adapters, [{a.a.shape[2]}] -> {a.parts}, are not of {shapes.get(name, 'qkv, o, gate_up or down')}")
    if len({a.a.shape[0] for ad in adapters for a in ad.values()}) > 1: raise ValueError(f"{what}: as many adapters in every block and projection (an adapter's number is the same in all)")
    return [dict(ad) for ad in adapters]

  @staticmethod
  def _check_of(what, of, n, adapters):
    """Each of n sequences' adapter, checked (None: none has one)."""
    if of is None: return np.full(n, -1, np.int64)
    of, count = np.asarray(of, np.int64), next((a.a.shape[0] for ad in adapters or () for a in ad.values()), 0)
    if of.shape != (n,): raise ValueError(f"{what}: {n} sequences' adapters")
    if ((of < -1) | (of >= count)).any(): raise ValueError(f"{what}: an adapter outside 0..{count - 1} (-1: none)" if count else f"{what}: an adapter where there are none")
    return of

  def step_pages(self, tokens, places, tables, page=64, adapters=None, of=None):
    """A step over sequences whose keys and values lie in pages of the cache (its slots * context rows cut into pages of `page`, 16, 32,
    64, ...), as many tokens of each as there are: whole prompts, chunks of them and single tokens in one call. Sequence i's tokens
    are at places places[i], places[i] + 1, ..., its place p in page tables[i][p // page]; sequences may begin with the same pages (a common
    prompt), but what rows are put into is one's own. The pages are the caller's to hand out, and so are the rows of slots that
    they lie in. adapters: for each block a dict of ops.Adapters, of any of "qkv" (parts q, k, v), "o", "gate_up" (gate, up) and "down", as many
    in each (one that leaves a projection alone has zeros there); of: each sequence's (-1: none). Returns each sequence's last token's logits ([n][vocab] fp32) and greedy picks ([n] int32), within the
    rounding of bf16 rows and fp32 sums of prefill's."""
    c, what = self.c, "step_pages"
    ops.attention_heads_ok(c.heads, c.kv, self.hd)
    n = len(tokens)
    lens = np.array([len(t) for t in tokens], np.int64)
    if n < 1 or (lens < 1).any(): raise ValueError(f"{what}: at least a token of each sequence")
    places = np.asarray(places, np.int64)
    tab = self._page_layout(what, places, lens, tables, page)
    adapters = self._check_adapters(what, adapters)
    of = self._check_of(what, of, n, adapters)
    T, starts = int(lens.sum()), np.concatenate([[0], np.cumsum(lens)])
    ints = np.concatenate([np.concatenate([np.asarray(t, np.int64) for t in tokens]), starts, places, starts[1:] - 1, np.repeat(of, lens), tab.reshape(-1)]).astype(np.int32)
    held = torch.empty(ints.size, dtype=torch.int32, device=self.device)
    if ints.size <= PUT_MAX: ops.put_i32(ints, held)
    else: held.copy_(torch.from_numpy(ints))
    ids, st, p0, last, rows_of, t = held.split([T, n + 1, n, n, T, tab.size])
    most = int((places + lens).max())
    ws = ops.attention_paged_workspace(T, n, c.heads, c.kv, self.hd, most, self.device)
    return self._page_rows(self._page_buffers(T, adapters), T, n, ids, st, p0, last, rows_of, t.view(n, -1), page, most, ws, adapters)

  def page_step(self, n, pages, page=64, adapters=None):
    """step_pages for n sequences of one token each with up to `pages` pages, captured once and replayed (PageStep)."""
    return PageStep(self, n, pages, page, adapters)

  def _last_rows(self, x, last, n):
    """The final norm and the output layer of rows `last` of x (bf16 rows on the matrix cores from three on): logits and picks."""
    c = self.c
    xl = ops.gather_rows(x, last)
    few = n < 3
    xl = ops.rms_rows(xl, self.norm, c.eps, c.centered, out_dtype=torch.float32 if few else torch.bfloat16)
    logits = torch.empty(n, c.vocab, dtype=torch.float32, device=self.device)
    parts = torch.empty(n, c.vocab // 16, dtype=torch.int64, device=self.device)
    (ops.gemv if few else ops.gemm)(xl, self.head, ops.epilogue(lib.EP_STORE, argmax_parts=parts), out=logits)
    return logits, ops.argmax_parts(parts)

  def step(self, ids=None, places=None, slots=None, replay=True):
    """One step: the logits (fp32, [batch][vocab]) and greedy picks for tokens ids at places: the model's own, before any rules
    (a row under rules takes its token from heads). With replay, the step runs as
    a HIP graph captured on the first call (every later step launches the same kernels: places are data)."""
    if ids is not None or places is not None: self._put(ids, places, slots)
    if not self.placed: raise ValueError("step: the rows' places are to be set again after share_prefix")
    if not replay:
      self._step()
    else:
      if self.graph is None:
        self._step()  # warm: every kernel loaded before capture
        torch.cuda.synchronize(self.device)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
          self._step()
        self.graph = g
      self.graph.replay()
    return self.logits, self.picks

  def advance(self):
    """Each row's next place and its pick as the next token, on the GPU (no host round trip): greedy decoding by the model's own
    logits. Rows under rules are stepped with the tokens drawn from heads(rules=) instead, step(tokens, places). Raises
    once a row's next place would pass the cache or RoPE's tables (the host keeps the largest place: set_rows', plus
    one a call)."""
    if self.top_own + 1 >= self.context or self.top + 1 >= self.c.places: raise ValueError(f"advance: place {self.top + 1} past the cache or RoPE's tables")
    self.top += 1
    self.top_own += 1
    self.ids.copy_(self.picks)
    self.places.add_(1)
    self.rows.add_(1)

  def heads(self, k=64, inv_temp=None, rules=None):
    """The last step's logit heads (models/serve.py:31-47): each row's k best logits and their tokens, and given each
    row's 1/temperature, the log of the sum of exp(x t) over its row (ops.logit_heads: fh_logit_heads). rules: ops.logit_rules'
    arguments (each request's penalties, biases and grammar mask), whose logits the heads are then of; the step's own logits and
    picks stay. A row whose mask leaves nothing has -inf for its values and its sum."""
    logits = self.logits
    if rules:
      if getattr(self, "_ruled", None) is None: self._ruled = torch.empty_like(self.logits)
      logits = ops.logit_rules(self.logits, out=self._ruled, **rules)
    if inv_temp is not None and not isinstance(inv_temp, torch.Tensor):
      inv_temp = torch.as_tensor(inv_temp, dtype=torch.float32, device=self.device).reshape(-1)
    return ops.logit_heads(logits, k, inv_temp)


class PageStep:
  """A decode step of `n` sequences over a Decoder's cache in pages (Decoder.page_step), replayed as one HIP graph: their tokens, places,
  pages and which adapter each has are data. The adapters themselves are those it was made with: others take a step of their own, or go into
  the same tensors in place. A sequence of the batch that nobody holds steps a page of its own."""

  def __init__(self, dec, n, pages, page, adapters):
    ops.attention_heads_ok(dec.c.heads, dec.c.kv, dec.hd)
    if n < 1 or pages < 1: raise ValueError("page_step: at least a sequence and a page")
    if page < 16 or page & (page - 1) or dec.slots * dec.part % page: raise ValueError(f"page_step: pages of 16, 32, 64, ... rows of a cache of {dec.slots * dec.part}")
    self.dec, self.n, self.pages, self.page, self.adapters, self.graph = dec, n, pages, page, dec._check_adapters("page_step", adapters), None
    c, dev = dec.c, dec.device
    self._int = torch.zeros(2 * n + n * pages + n, dtype=torch.int32, device=dev)
    self.ids, self.p0, self.of, self.tables = self._int.split([n, n, n, n * pages])
    self.tables = self.tables.view(n, pages).fill_(-1)  # (a step before any set puts nothing into the cache)
    self.starts = torch.arange(n + 1, dtype=torch.int32, device=dev)
    self.bufs = dec._page_buffers(n, self.adapters)
    self.ws = ops.attention_paged_workspace(n, n, c.heads, c.kv, dec.hd, pages * page, dev)

  def _step(self):
    return self.dec._page_rows(self.bufs, self.n, self.n, self.ids, self.starts, self.p0, self.starts[:self.n], self.of, self.tables, self.page,
                               self.pages * self.page, self.ws, self.adapters)

  def set(self, tokens, places, tables, of=None):
    """The sequences' next tokens (the host's, or integers on the GPU as they are: a step's own picks), places and pages, and their
    adapters (-1, or none given: none)."""
    n = self.n
    places = np.asarray(places, np.int64)
    tab = self.dec._page_layout("page_step", places, np.ones(n, np.int64), tables, self.page)
    if tab.shape[1] > self.pages: raise ValueError(f"page_step: up to {self.pages} pages a sequence, not {tab.shape[1]}")
    there = torch.is_tensor(tokens) and tokens.is_cuda
    if there and tokens.dtype not in (torch.int32, torch.int64): raise ValueError(f"page_step: tokens are integers, not {tokens.dtype}")
    if not there: tokens = np.asarray(tokens, np.int64)
    if tokens.shape != (n,): raise ValueError(f"page_step: {n} tokens, not {tuple(tokens.shape)}")
    of = self.dec._check_of("page_step", of, n, self.adapters)
    wide = np.full((n, self.pages), -1, np.int64)
    wide[:, :tab.shape[1]] = tab
    ints = np.concatenate(([] if there else [tokens]) + [places, of, wide.reshape(-1)]).astype(np.int32)
    held = self._int[n:] if there else self._int
    if ints.size <= PUT_MAX: ops.put_i32(ints, held)
    else: held.copy_(torch.from_numpy(ints))
    if there: self.ids.copy_(tokens)

  def step(self, tokens=None, places=None, tables=None, of=None, replay=True):
    """One step: the logits ([n][vocab] fp32) and greedy picks ([n] int32); a replayed step's are the graph's, as they are until the
    next."""
    if tokens is not None: self.set(tokens, places, tables, of)
    if not replay: return self._step()
    if self.graph is None:
      self._step()  # warm: every kernel loaded before capture
      torch.cuda.synchronize(self.dec.device)
      g = torch.cuda.CUDAGraph()
      with torch.cuda.graph(g): self.out = self._step()
      self.graph = g
    self.graph.replay()
    return self.out


def numpy_weights(w):
  """weights(name, shape) over a dict of numpy arrays (bf16 values as float32), for Decoder."""
  def get(name, shape):
    a = np.asarray(w[name], np.float32).reshape(shape)
    return torch.from_numpy(np.ascontiguousarray(a))
  return get


def random_weights(c, seed=0, sd=0.02, norm_sd=0.1, embed_sd=1.0, device="cuda"):
  """weights(name, shape) drawn on the GPU: matrices N(0, sd), norms N(1, norm_sd), the embedding N(0, embed_sd), each
  rounded to bf16, from a generator seeded by seed and the weight's name (so each is the same whatever asks first)."""
  def get(name, shape):
    g = torch.Generator(device=device)
    g.manual_seed(seed * 1000003 + sum(ord(ch) * 31 ** i for i, ch in enumerate(name)) % (2**31))
    if "norm" in name: t = torch.randn(*shape, generator=g, device=device) * norm_sd + 1
    elif name == "embed": t = torch.randn(*shape, generator=g, device=device) * embed_sd
    else: t = torch.randn(*shape, generator=g, device=device) * sd
    return t.to(torch.bfloat16)
  return get
