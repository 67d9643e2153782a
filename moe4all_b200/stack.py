"""A stack of layers as the graph builder emits them for a step
(crates/infr-llama/src/seam/runner.rs:7999-8176; layer shape pinned in
crates/infr-core/src/fusion.rs:735-737): MoE FFN sub-layers, and with `attn` an attention sub-layer ahead of each:

    hn     = RmsNorm(hidden, a_l, eps)                  with attn
    qkv    = Linear(hn, wqkv_l)
    q      = RopeKv(qkv) -> k, v into layer l's pages
    hidden = Add(hidden, Linear(Attention(q), wo_l))

    hn     = RmsNorm(hidden, w_l, eps)
    sub    = MoeFfn(hn) (+ shared expert)
    hidden = Add(hidden, sub)

With `ends` the step goes from tokens to tokens: Embed writes `hidden` ahead of the layers, and behind them

    hn     = RmsNorm(hidden, w, eps)
    logits = Linear(hn, head)
    tokens = Sample(logits)

Every op goes through the C ABI; the whole step can be recorded once and replayed
(`Backend::compile` + decode replay)."""
from __future__ import annotations

import weakref
from dataclasses import dataclass, field
from typing import List, Optional

import torch

from .backend import Attention, Buffer, CudaBackend, DType, Embed, MoeFfn, RopeKv, Sample


@dataclass
class AttnWeights:
    """One layer's attention: the norm ahead of it, q / k / v in one projection [(n_head + 2 n_kv) head_dim, ne], the output
    projection [ne, n_head head_dim], both of `dtype`, and the per-head norms of q and k where the model has them."""
    norm: torch.Tensor
    wqkv: Buffer
    wo: Buffer
    q_norm: Optional[torch.Tensor] = None
    k_norm: Optional[torch.Tensor] = None
    dtype: DType = DType.F32


@dataclass
class StackAttention:
    """The attention of a `MoeStack` over pages that all of its layers address alike: sequence s has kv_len[s] tokens with the step's new
    ones, which are the stack's rows cu_q[s] .. cu_q[s + 1] - 1.  The three arrays are i32 tensors on the device, read when a step runs: a
    recorded step follows new lengths and pages written into them.  `caches[l]` are layer l's (k, v), f16 [n_pages, n_kv, page_size, head_dim], or, of 8 bits,
    its (k, v, k_scale, v_scale): codes, uint8 of that shape, and a scale to each 16 of them, uint8 [n_pages, n_kv, page_size, head_dim / 16].

    Several stacks may have the same one (a stack of prompt chunks and one of single tokens over the same caches): weights, caches and arrays are
    shared, the rows between the ops are each stack's own."""
    layers: List[AttnWeights]
    n_head: int
    n_kv: int
    head_dim: int
    cu_q: torch.Tensor
    kv_len: torch.Tensor
    page_table: torch.Tensor
    page_size: int
    caches: List[tuple]
    max_q: int = 0  # longest sequence of new rows, as far as known (1 for a decode step): picks the kernel
    window: int = 0
    rope_base: float = 1e4
    n_rot: Optional[int] = None  # whole heads unless given
    interleaved: bool = False
    _bound: weakref.WeakSet = field(default_factory=weakref.WeakSet, init=False, repr=False, compare=False)

    def bind(self, be: CudaBackend, rows: int, ne: int, eps: float, hidden: Buffer, device) -> "BoundAttention":
        """These layers on a stack's rows: the ops, and buffers of the stack's own between them."""
        bound = BoundAttention(self, be, rows, ne, eps, hidden, device)
        self._bound.add(bound)
        return bound

    def layer(self, li: int) -> None:
        """One attention sub-layer in place on the `hidden` of the stack that this is bound to, where there is one."""
        bound = list(self._bound)
        if len(bound) != 1:
            raise RuntimeError(f"StackAttention.layer: bound to {len(bound)} stacks: call the stack's attn_layer")
        bound[0].layer(li)


class BoundAttention:
    """A `StackAttention` on the rows of one stack: buffers between the ops, and the ops over them."""

    def __init__(self, attn: StackAttention, be: CudaBackend, rows: int, ne: int, eps: float, hidden: Buffer, device):
        H, K, hd = attn.n_head, attn.n_kv, attn.head_dim
        # (the library sees addresses and bytes: types and shapes are seen here or not at all)
        n_seq = attn.kv_len.numel()
        for name, t in (("cu_q", attn.cu_q), ("kv_len", attn.kv_len), ("page_table", attn.page_table)):
            if t.dtype != torch.int32:
                raise ValueError(f"StackAttention.{name} must be int32, not {t.dtype}")
        if attn.cu_q.numel() != n_seq + 1 or attn.page_table.dim() != 2 or attn.page_table.shape[0] != n_seq:
            raise ValueError("StackAttention: cu_q is [n_seq + 1], kv_len [n_seq], page_table [n_seq, max_pages]")
        if len(attn.layers) != len(attn.caches) or not attn.layers:
            raise ValueError("StackAttention: a (k, v) pair of caches for each layer")
        shape = (attn.caches[0][0].shape[0], K, attn.page_size, hd)
        scales = (*shape[:3], hd // 16)
        for kv in attn.caches:
            if len(kv) not in (2, 4):
                raise ValueError(f"StackAttention: a layer's caches are (k, v) or, of 8 bits, (k, v, k_scale, v_scale), not {len(kv)} tensors")
            for c in kv[:2] if len(kv) == 2 else ():
                if c.dtype != torch.float16 or tuple(c.shape) != shape:
                    raise ValueError(f"StackAttention: caches are float16 [n_pages, n_kv, page_size, head_dim], {shape} here, not {c.dtype} {tuple(c.shape)}")
            for c, want in zip(kv, (shape, shape, scales, scales)) if len(kv) == 4 else ():
                if c.dtype != torch.uint8 or tuple(c.shape) != want:
                    raise ValueError(f"StackAttention: caches of 8 bits are uint8, codes {shape} and scales {scales} here, not {c.dtype} {tuple(c.shape)}")
        wide, w = (H + 2 * K) * hd, be.wrap_tensor
        self._be, self._layers, self._shape, self._hidden = be, attn.layers, (rows, ne, eps, wide, H * hd), hidden
        self._rows = [torch.zeros(rows, n, device=device) for n in (ne, wide, H * hd, H * hd, ne)]
        self._hn, self._qkv, q, out, self._sub = (w(t) for t in self._rows)
        self._out = out
        # (the parts of the wide rows: their memory is _rows')
        part = lambda first: be.wrap(self._rows[1].data_ptr() + 4 * first, 4 * (rows * wide - first))
        batch = dict(cu_q=w(attn.cu_q), kv_len=w(attn.kv_len), page_table=w(attn.page_table), rows=rows, n_seq=n_seq, n_head=H, n_kv=K,
                     head_dim=hd, n_pages=shape[0], page_size=attn.page_size, max_pages=attn.page_table.shape[1])
        parts = part(0), part(H * hd), part((H + K) * hd)
        self._ops = []
        for L, kv in zip(attn.layers, attn.caches):
            opt = lambda t: None if t is None else w(t)
            kc, vc = w(kv[0]), w(kv[1])
            bits8 = dict(k_scale=w(kv[2]), v_scale=w(kv[3])) if len(kv) == 4 else {}
            self._ops.append((w(L.norm), RopeKv(q=parts[0], k=parts[1], v=parts[2], q_stride=wide, k_stride=wide, v_stride=wide, q_out=q, k_cache=kc, v_cache=vc,
                                                n_rot=hd if attn.n_rot is None else attn.n_rot, interleaved=attn.interleaved, rope_base=attn.rope_base,
                                                q_norm=opt(L.q_norm), k_norm=opt(L.k_norm), norm_eps=eps, **bits8, **batch),
                              Attention(q=q, k=kc, v=vc, out=out, scale=hd ** -0.5, max_q=attn.max_q, window=attn.window, **bits8, **batch)))

    def layer(self, li: int) -> None:
        """One attention sub-layer in place on `hidden`."""
        be, L, (norm, rope, attention) = self._be, self._layers[li], self._ops[li]
        rows, ne, eps, wide, n_out = self._shape
        be.rms_norm(self._hidden, norm, self._hn, rows, ne, eps)
        be.linear(L.dtype, L.wqkv, self._hn, self._qkv, rows, ne, wide)
        be.rope_kv(rope)
        be.attention(attention)
        be.linear(L.dtype, L.wo, self._out, self._sub, rows, n_out, ne)
        be.add(self._hidden, self._sub, self._hidden, rows * ne)


@dataclass
class StackEnds:
    """What stands ahead of the layers and behind them.  `tokens` is an i32 tensor on the device of the rows' ids, read when a step runs.  Without a `head` the
    step ends with the last layer: a stack of prompt chunks, whose last token is the first step's of a stack with one.  With it every row is answered: the
    token sampled by `u` (f32, a random number in [0, 1) to each row, read when a step runs) takes its place in `tokens`, so that a recorded step goes on from
    its own answer.  Settings are tensors of a number to each row, as `Sample` has them: temperature, top_p and min_p f32, top_k i32."""
    table: Buffer  # [n_vocab, ne] of table_dtype
    tokens: torch.Tensor
    n_vocab: int
    table_dtype: DType = DType.F32
    scale: float = 1.0  # of the table's rows
    norm: Optional[torch.Tensor] = None  # [ne] f32
    head: Optional[Buffer] = None  # [n_vocab, ne] of head_dtype: F32 or a block format, as a Linear has it
    head_dtype: DType = DType.F32
    u: Optional[torch.Tensor] = None
    temperature: Optional[torch.Tensor] = None
    top_k: Optional[torch.Tensor] = None
    top_p: Optional[torch.Tensor] = None
    min_p: Optional[torch.Tensor] = None


class BoundEnds:
    """`StackEnds` on the rows of one stack."""

    def __init__(self, ends: StackEnds, be: CudaBackend, rows: int, ne: int, eps: float, hidden: Buffer, hn: Buffer, device):
        settings = {n: getattr(ends, n) for n in ("temperature", "top_k", "top_p", "min_p") if getattr(ends, n) is not None}
        for name, t, want in [("tokens", ends.tokens, torch.int32)] + [(n, t, torch.int32 if n == "top_k" else torch.float32) for n, t in (("u", ends.u), *settings.items()) if t is not None]:
            if t.dtype != want or t.numel() != rows or not t.is_contiguous():
                raise ValueError(f"StackEnds.{name} is {want} of the {rows} rows, not {t.dtype} {tuple(t.shape)}")
        if ends.head is not None and (ends.norm is None or ends.u is None):
            raise ValueError("StackEnds: a head needs the norm ahead of it, and random numbers")
        if ends.norm is not None and (ends.norm.dtype != torch.float32 or ends.norm.numel() != ne or not ends.norm.is_contiguous()):
            raise ValueError(f"StackEnds.norm is float32 of the {ne} values of a row, not {ends.norm.dtype} {tuple(ends.norm.shape)}")
        if ends.head is not None and DType(ends.head_dtype) in (DType.F16, DType.BF16):
            raise ValueError(f"StackEnds.head_dtype: a Linear has no weights of 16 bits ({DType(ends.head_dtype).name}): F32 or a block format")
        if ends.head is None and (ends.u is not None or settings):
            raise ValueError("StackEnds: without a head nothing is sampled")
        w = be.wrap_tensor
        self._be, self._rows, self._ne, self._eps, self._hidden, self._hn, self._ends = be, rows, ne, eps, hidden, hn, ends
        tokens = w(ends.tokens)
        self._embed = Embed(table=ends.table, ids=tokens, dst=hidden, rows=rows, ne=ne, n_vocab=ends.n_vocab, dtype=ends.table_dtype, scale=ends.scale)
        self._sample = None
        if ends.head is not None:
            self.logits = torch.zeros(rows, ends.n_vocab, device=device)
            self._norm = w(ends.norm)
            self._sample = Sample(logits=w(self.logits), u=w(ends.u), ids=tokens, rows=rows, n_vocab=ends.n_vocab, **{n: w(t) for n, t in settings.items()})

    def embed(self) -> None:
        self._be.embed(self._embed)

    def answer(self) -> None:
        if self._sample is None:
            return
        be, ends = self._be, self._ends
        be.rms_norm(self._hidden, self._norm, self._hn, self._rows, self._ne, self._eps)
        be.linear(ends.head_dtype, ends.head, self._hn, self._sample.logits, self._rows, self._ne, ends.n_vocab)
        be.sample(self._sample)


class MoeStack:
    def __init__(self, be: CudaBackend, layers: List, norm_weights: List[torch.Tensor], rows: int, ne: int, n_expert: int,
                 n_used: int, n_ff: int, sh_ff: int = 0, eps: float = 1e-6, fused: bool = True, attn: Optional[StackAttention] = None,
                 ends: Optional[StackEnds] = None, **route_kw):
        """fused: fold RmsNorm and the residual Add into the MoE op (the reference's
        RmsNorm->MoeFfn and MoeFfn->Add peepholes, crates/infr-core/src/fusion.rs:17-25) instead of
        running them as kernels of their own.  attn: an attention sub-layer ahead of every MoE one.  ends: a step begins
        with tokens and, where they have a head, ends with tokens."""
        assert len(layers) == len(norm_weights)
        self.be, self.layers, self.rows, self.ne, self.eps = be, layers, rows, ne, eps
        dev = norm_weights[0].device
        self.hidden = torch.zeros(rows, ne, device=dev)
        self.hn = torch.zeros(rows, ne, device=dev)
        self.sub = torch.zeros(rows, ne, device=dev)
        # each layer's ids on a 16-byte boundary, as the library wants its buffers
        per_layer = (rows * n_used + 3) // 4 * 4
        self.ids = torch.zeros(len(layers), per_layer, dtype=torch.int32, device=dev)[:, : rows * n_used].unflatten(1, (rows, n_used))
        self._nw = norm_weights
        self.b_hidden, self.b_hn, self.b_sub = be.wrap_tensor(self.hidden), be.wrap_tensor(self.hn), be.wrap_tensor(self.sub)
        self.b_nw = [be.wrap_tensor(w) for w in norm_weights]
        self.fused = fused
        self.ops = []
        for li, L in enumerate(layers):
            b = L.b
            fuse = dict(x=self.b_hidden, dst=self.b_hidden, norm_weight=self.b_nw[li], norm_eps=eps, residual=self.b_hidden) \
                if fused else dict(x=self.b_hn, dst=self.b_sub)
            self.ops.append(MoeFfn(router=b["router"], gate_exps=b["gate"], up_exps=b["up"], down_exps=b["down"],
                                   rows=rows, ne=ne, n_expert=n_expert, n_used=n_used, n_ff_exp=n_ff,
                                   ids_out=be.wrap_tensor(self.ids[li]), sh_gate=b.get("sh_gate"), sh_up=b.get("sh_up"),
                                   sh_down=b.get("sh_down"), sh_gate_inp=b.get("sh_gate_inp"),
                                   sh_ff=sh_ff if "sh_gate" in b else 0, **fuse, **route_kw))
        self.plan = None
        if attn is not None and len(attn.layers) != len(layers):
            raise ValueError(f"MoeStack: {len(layers)} layers, and attention for {len(attn.layers)}")
        self.attn = attn
        self._attn = None if attn is None else attn.bind(be, rows, ne, eps, self.b_hidden, dev)
        self.ends = None if ends is None else BoundEnds(ends, be, rows, ne, eps, self.b_hidden, self.b_hn, dev)
        if dev.type == "cuda":
            # The buffers above are torch's, in the order of its stream: they may still be somebody else's there, and their zeros on the way.  The first step's ops
            # run on the backend's.
            torch.cuda.current_stream(dev).synchronize()

    def attn_layer(self, li: int) -> None:
        """The attention sub-layer of one layer in place on `hidden`."""
        self._attn.layer(li)

    def layer(self, li: int) -> None:
        """One layer in place on `hidden`."""
        be = self.be
        if self._attn is not None:
            self._attn.layer(li)
        if self.fused:
            be.moe_ffn(self.ops[li])
            return
        be.rms_norm(self.b_hidden, self.b_nw[li], self.b_hn, self.rows, self.ne, self.eps)
        be.moe_ffn(self.ops[li])
        be.add(self.b_hidden, self.b_sub, self.b_hidden, self.rows * self.ne)

    def step(self) -> None:
        if self.ends is not None:
            self.ends.embed()
        for li in range(len(self.layers)):
            self.layer(li)
        if self.ends is not None:
            self.ends.answer()

    def record(self) -> None:
        """Records a step for `replay`.  Runs one first, on what `hidden` holds: with attention it writes keys and values into the caller's pages, as any step
        does (of the tokens that kv_len and cu_q say; the step that is replayed for these writes the same places), and with a
        head it leaves its answers in `tokens`: write the first replay's there after it."""
        self.step()  # scratch sized, kernels loaded
        self.be.sync()
        self.be.graph_begin()
        self.step()
        self.plan = self.be.graph_end()

    def replay(self) -> None:
        self.be.execute(self.plan)
