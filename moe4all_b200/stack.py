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

Every op goes through the C ABI; the whole step can be recorded once and replayed
(`Backend::compile` + decode replay)."""
from __future__ import annotations

import weakref
from dataclasses import dataclass, field
from typing import List, Optional

import torch

from .backend import Attention, Buffer, CudaBackend, DType, MoeFfn, RopeKv


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
    recorded step follows new lengths and pages written into them.  `caches[l]` are layer l's (k, v), f16 [n_pages, n_kv, page_size, head_dim].

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
        for c in (c for kv in attn.caches for c in kv):
            if c.dtype != torch.float16 or tuple(c.shape) != shape:
                raise ValueError(f"StackAttention: caches are float16 [n_pages, n_kv, page_size, head_dim], {shape} here, not {c.dtype} {tuple(c.shape)}")
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
        for L, (k, v) in zip(attn.layers, attn.caches):
            opt = lambda t: None if t is None else w(t)
            kc, vc = w(k), w(v)
            self._ops.append((w(L.norm), RopeKv(q=parts[0], k=parts[1], v=parts[2], q_stride=wide, k_stride=wide, v_stride=wide, q_out=q, k_cache=kc, v_cache=vc,
                                                n_rot=hd if attn.n_rot is None else attn.n_rot, interleaved=attn.interleaved, rope_base=attn.rope_base,
                                                q_norm=opt(L.q_norm), k_norm=opt(L.k_norm), norm_eps=eps, **batch),
                              Attention(q=q, k=kc, v=vc, out=out, scale=hd ** -0.5, max_q=attn.max_q, window=attn.window, **batch)))

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


class MoeStack:
    def __init__(self, be: CudaBackend, layers: List, norm_weights: List[torch.Tensor], rows: int, ne: int, n_expert: int,
                 n_used: int, n_ff: int, sh_ff: int = 0, eps: float = 1e-6, fused: bool = True, attn: Optional[StackAttention] = None, **route_kw):
        """fused: fold RmsNorm and the residual Add into the MoE op (the reference's
        RmsNorm->MoeFfn and MoeFfn->Add peepholes, crates/infr-core/src/fusion.rs:17-25) instead of
        running them as kernels of their own.  attn: an attention sub-layer ahead of every MoE one."""
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
        for li in range(len(self.layers)):
            self.layer(li)

    def record(self) -> None:
        """Records a step for `replay`.  Runs one first, on what `hidden` holds: with attention it writes keys and values into the caller's pages, as any step
        does (of the tokens that kv_len and cu_q say; the step that is replayed for these writes the same places)."""
        self.step()  # scratch sized, kernels loaded
        self.be.sync()
        self.be.graph_begin()
        self.step()
        self.plan = self.be.graph_end()

    def replay(self) -> None:
        self.be.execute(self.plan)
