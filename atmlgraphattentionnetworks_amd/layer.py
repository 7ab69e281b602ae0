"""Drop-in ``GraphAttentionLayer`` for ``GAT.py:6-67`` on MI355X.

Same constructor signature, attributes, parameter init order and
``state_dict`` keys as the reference (``GAT.py:8-35``), so ``GATNet.py`` and
the ``run_*.py`` scripts construct, checkpoint and call it unchanged.  The
forward (``GAT.py:37-67``) runs entirely in the HIP library:

  1. CSR by target with appended self-loops, cached per ``edge_index``
     (``graph.get_csr``; replaces ``add_self_loops``, ``GAT.py:38``);
  2. ``gat_project``: one fp32 MFMA GEMM for all heads with the attention
     Linears fused (replaces the head loop, ``GAT.py:42-52``);
  3. ``gat_edge_aggregate``: scores, LeakyReLU, segmented softmax,
     weighted aggregation, concat / head-mean, bias (``GAT.py:53-67``).

When autograd needs the result, or in training mode with dropout > 0, the
forward goes through ``training.GATFunction`` instead: the same two kernels
plus attention dropout (``GAT.py:61``) and a HIP backward pass.

No PyG import, no CPU path: a CPU tensor or a missing library raises.
"""
from __future__ import annotations

import collections
import itertools
import weakref
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib, tuning
from .graph import CSRGraph, get_csr, rotated_col, sched_csr

__all__ = ["GraphAttentionLayer", "GraphAttentionLayerActivationTest", "score_activation_code",
           "PackedParams", "pack_params", "gat_forward", "ForwardPlan", "wh_slices", "NodeTable",
           "alloc_table", "project", "edge_aggregate"]


def refuse_tangents(what: str, *tensors: torch.Tensor) -> None:
    """The kernels have a backward and no forward-mode derivative.  They read a dual
    tensor's values only, so its tangent would be lost without a word."""
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None
           for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def refuse_recording(what: str, jit: bool = False) -> None:
    """What records torch's operations does not see the library write into its outputs: a
    recorded call would give whatever the memory held.  ``jit``: the caller has no form that
    ``torch.jit.trace`` can keep either (an autograd function is kept as a whole)."""
    if torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None or \
            (jit and torch._C._is_tracing()):
        raise RuntimeError(f"{what} cannot be recorded: its kernels are outside torch's operators")


class PackedParams:
    """Device buffers derived from the per-head ``Linear`` parameters (never
    stored in the state_dict; rebuilt when any parameter's version moves)."""

    __slots__ = ("w", "b", "a_src", "c_src", "a_dst", "c_dst", "key")

    def __init__(self, w, b, a_src, c_src, a_dst, c_dst, key):
        self.w, self.b = w, b
        self.a_src, self.c_src, self.a_dst, self.c_dst = a_src, c_src, a_dst, c_dst
        self.key = key


def _param_list(layer: "GraphAttentionLayer"):
    """The 6H packed parameters, read through ``_parameters`` (Module.__getattr__
    costs ~1 us per access, the dominant host cost of a small forward)."""
    out = []
    for mods in (layer.ws, layer.attentions1, layer.attentions2):
        ms = list(mods._modules.values())
        out.extend(m._parameters["weight"] for m in ms)
        out.extend(m._parameters["bias"] for m in ms)
    return out


def _param_key(params) -> Tuple:
    return tuple([p._version for p in params] + [p.data_ptr() for p in params])


def pack_params(layer: "GraphAttentionLayer", cached: Optional[PackedParams] = None) -> PackedParams:
    params = _param_list(layer)
    key = _param_key(params)
    if cached is not None and cached.key == key:
        return cached
    H = layer.num_heads
    with torch.no_grad():
        w = torch.cat(params[0:H], 0).contiguous()  # [H*F, Fin]
        b = torch.cat(params[H:2 * H], 0).contiguous()  # [H*F]
        a_src = torch.cat([p.reshape(-1) for p in params[2 * H:3 * H]]).contiguous()
        c_src = torch.cat([p.reshape(-1) for p in params[3 * H:4 * H]]).contiguous()
        a_dst = torch.cat([p.reshape(-1) for p in params[4 * H:5 * H]]).contiguous()
        c_dst = torch.cat([p.reshape(-1) for p in params[5 * H:6 * H]]).contiguous()
    return PackedParams(w, b, a_src, c_src, a_dst, c_dst, key)


# Packed-buffer invalidation without walking the 6H parameters per forward
# (that walk cost ~16 us of host time per call).  Each per-head Linear carries
# its layer's token; a global parameter-registration hook marks the layer
# stale when one of them gets a new Parameter (setattr, load_state_dict with
# assign=True).  packed() also checks that the first head's parameters still
# alias the packed buffers, which catches .to()/deepcopy-style re-storage.
_owners: "weakref.WeakValueDictionary[int, torch.nn.Module]" = weakref.WeakValueDictionary()
_tokens = itertools.count(1)


def _mark_owner_dirty(module, name, param):
    token = module.__dict__.get("_gat_owner")
    if token is not None:
        owner = _owners.get(token)
        if owner is not None:
            owner.__dict__["_packed_dirty"] = True
    return None


torch.nn.modules.module.register_module_parameter_registration_hook(_mark_owner_dirty)


def _stream(device: torch.device) -> int:
    """Raw hipStream_t of torch's current stream on ``device``."""
    return torch._C._cuda_getCurrentRawStream(device.index)


class NodeTable(NamedTuple):
    """Per-source-node outputs of the projection, as the edge kernel reads
    them: Wh rows (stride ld_wh floats) and s_src (stride ld_s floats).

    Default layout: Wh [N, round_up(H*F, 4)] and a compact s_src [N, H].
    Packed layout (``packed=True``): one buffer [N, ld] holding both (one
    collective moves both; see distributed.py), ``buf`` is that buffer.
    Wh-only layout (``wh_only=True``): ``s_src`` is None — for shapes whose
    edge kernel recomputes s_src from the gathered Wh row (the library then
    refuses, rather than guesses, if it would need s_src).
    Sliced layout (``slices > 1``): Wh as ``slices`` column planes
    [slices, N, ld_wh = H*F/slices] (gat_project_sliced / gat_edge_aggregate_sliced);
    no s_src (the sliced edge kernel recomputes it).  ``rows`` views keep the
    plane stride (``wh.stride(0)``), so a rank can project into its slot."""
    wh: torch.Tensor
    ld_wh: int
    s_src: Optional[torch.Tensor]
    ld_s: int
    buf: Optional[torch.Tensor] = None
    slices: int = 1

    def rows(self, start: int, stop: int) -> "NodeTable":
        """The table restricted to rows [start, stop) (views, same strides)."""
        if self.slices > 1:
            return NodeTable(self.wh[:, start:stop], self.ld_wh, None, self.ld_s, None,
                             self.slices)
        return NodeTable(self.wh[start:stop], self.ld_wh,
                         None if self.s_src is None else self.s_src[start:stop], self.ld_s,
                         None if self.buf is None else self.buf[start:stop])


def alloc_table(n: int, heads: int, f: int, device, packed: bool = False,
                wh_only: bool = False, slices: int = 1) -> NodeTable:
    if slices > 1:
        if packed or (heads * f) % slices:
            raise ValueError("a sliced table is Wh planes only")
        sw = heads * f // slices
        wh = torch.zeros(slices, n, sw, dtype=torch.float32, device=device)
        return NodeTable(wh, sw, None, heads, wh, slices)
    if wh_only:
        hfp = (heads * f + 3) // 4 * 4
        buf = torch.zeros(n, hfp, dtype=torch.float32, device=device)
        return NodeTable(buf, hfp, None, heads, buf)
    if packed:
        ld, s_off = _lib.table_layout(heads, f)
        buf = torch.zeros(n, ld, dtype=torch.float32, device=device)
        return NodeTable(buf, ld, buf[:, s_off:], ld, buf)
    hfp = (heads * f + 3) // 4 * 4
    wh = torch.empty(n, hfp, dtype=torch.float32, device=device)
    s_src = torch.empty(n, heads, dtype=torch.float32, device=device)
    return NodeTable(wh, hfp, s_src, heads)


def project_workspace(device, fin: int, heads: int, f: int) -> Optional[torch.Tensor]:
    """The optional workspace of ``gat_project_ex`` (Fin > 128: W split into
    bf16 planes once per launch instead of in every workgroup), or None."""
    nb = _lib.project_workspace_bytes(fin, heads, f)
    return torch.empty(nb, dtype=torch.uint8, device=device) if nb > 0 else None


def project(x: torch.Tensor, pp: PackedParams, heads: int, f: int,
            table: Optional[NodeTable] = None, s_dst: Optional[torch.Tensor] = None):
    """``gat_project_ex``: node table (Wh, s_src) and s_dst [N, H]."""
    lib = _lib.load()
    n, fin = x.shape
    if table is None:
        table = alloc_table(n, heads, f, x.device)
    if s_dst is None:
        s_dst = torch.empty(n, heads, dtype=torch.float32, device=x.device)
    ws = project_workspace(x.device, fin, heads, f)
    wsa = (0, 0) if ws is None else (ws.data_ptr(), ws.numel())
    args = (x.data_ptr(), n, fin, pp.w.data_ptr(), pp.b.data_ptr(), pp.a_src.data_ptr(),
            pp.c_src.data_ptr(), pp.a_dst.data_ptr(), pp.c_dst.data_ptr(), heads, f)
    if table.slices > 1:
        # planes of wh.stride(0) / ld_wh rows; wh may be a rank's slot (rows view)
        _lib.check(lib.gat_project_ex(*args, table.slices, table.wh.data_ptr(),
                                      table.wh.stride(0) // table.ld_wh, 0, heads,
                                      s_dst.data_ptr(), 0, 0, *wsa, _stream(x.device)),
                   "gat_project_ex (planes)")
        return table, s_dst
    s_src = table.s_src
    if s_src is None:  # Wh-only table: the scores still have to go somewhere
        s_src = torch.empty(n, heads, dtype=torch.float32, device=x.device)
    _lib.check(lib.gat_project_ex(*args, 1, table.wh.data_ptr(), table.ld_wh, s_src.data_ptr(),
                                  heads if table.s_src is None else table.ld_s,
                                  s_dst.data_ptr(), 0, 0, *wsa, _stream(x.device)),
               "gat_project_ex")
    return table, s_dst


def edge_aggregate(csr, table: NodeTable, s_dst: torch.Tensor, heads: int, f: int,
                   concat: bool, bias: torch.Tensor, negative_slope: float = 0.2,
                   row_begin: int = 0, row_end: Optional[int] = None,
                   out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                   pp: Optional[PackedParams] = None):
    """``gat_edge_aggregate`` over target rows [row_begin, row_end).  With
    ``pp`` the library may recompute the source score from the gathered Wh
    row (a_src/c_src) instead of gathering s_src."""
    lib = _lib.load()
    rows = csr.num_nodes if row_end is None else row_end
    width = heads * f if concat else f
    if out is None:
        out = torch.empty(rows, width, dtype=torch.float32, device=table.wh.device)
    order = getattr(csr, "order", None)
    hint = csr.kernel_hint() if hasattr(csr, "kernel_hint") else \
        csr.num_edges // max(csr.num_nodes, 1)
    if table.slices > 1:
        if pp is None or lse is not None:
            raise ValueError("the sliced edge kernel recomputes s_src (pp) and has no lse")
        _lib.check(lib.gat_edge_aggregate_sliced(
            csr.rowptr.data_ptr(), csr.col.data_ptr(), 0 if order is None else order.data_ptr(),
            row_begin, rows, table.wh.data_ptr(), table.wh.stride(0) // table.ld_wh, table.slices,
            pp.a_src.data_ptr(), pp.c_src.data_ptr(), s_dst.data_ptr(), heads, f,
            float(negative_slope), bias.data_ptr(), out.data_ptr(), hint,
            _stream(table.wh.device)), "gat_edge_aggregate_sliced")
        return out
    _lib.check(lib.gat_edge_aggregate(
        csr.rowptr.data_ptr(), csr.col.data_ptr(), 0 if order is None else order.data_ptr(),
        row_begin, rows, table.wh.data_ptr(), table.ld_wh,
        0 if table.s_src is None else table.s_src.data_ptr(), table.ld_s,
        0 if pp is None else pp.a_src.data_ptr(), 0 if pp is None else pp.c_src.data_ptr(),
        s_dst.data_ptr(), heads, f, int(concat), float(negative_slope), bias.data_ptr(),
        out.data_ptr(), 0 if lse is None else lse.data_ptr(), hint, _stream(table.wh.device)),
        "gat_edge_aggregate")
    return out


def wh_slices(heads: int, f: int, concat: bool, negative_slope: float,
              edges_per_row: int = 0) -> int:
    """Number of column planes for the eval forward's node table
    (``gat_project_sliced`` / ``gat_edge_aggregate_sliced``), 1 = row-major.

    A plane holds whole heads; the edge kernel needs concat, LeakyReLU with
    slope in [0, 1] and f/4 a power of two.  Default: 128-byte plane rows (one
    cache line per gathered row, HF = 64 -> 2 planes) once rows average >= 16
    in-edges.  Measured with ``tools/slice_probe.py`` (interleaved, graph
    replay): edge kernel PPI 33.9 -> 30.0 us, Reddit scale 3.21 -> 2.49 ms;
    planes of 64 or 32 B rows are slower than row-major (more cache lines per
    wave instruction), and at ogbn-arxiv's 8 edges per row 2 planes lose
    (56.6 -> 61.8 us: each plane re-reads the row's indices and bookkeeping).
    ``GAT_WH_SLICES`` (A/B knob) overrides the default."""
    hf = heads * f
    env = tuning.get("GAT_WH_SLICES")
    if env is not None:
        s = int(env)
    elif hf % _PLANE_COLS == 0 and edges_per_row >= _MIN_SLICED_EPR:
        s = hf // _PLANE_COLS
    else:
        s = 1
    if s <= 1 or not concat or not (0.0 <= negative_slope <= 1.0):
        return 1
    if f % 4 or (f // 4) & (f // 4 - 1):
        return 1
    while s > 1 and (heads % s or (hf // s) % 4):
        s -= 1
    return max(s, 1)


_PLANE_COLS = 32        # 128-byte plane rows
_MIN_SLICED_EPR = 16    # average in-edges per row below which row-major wins


def fused_score_ok(heads: int, f: int, negative_slope: float) -> bool:
    """Shapes the fused-score edge kernels take (the source score recomputed
    from the gathered Wh row): LeakyReLU slope in [0, 1], f % 4 == 0 and f/4 a
    power of two."""
    hl = f // 4
    return 0.0 <= negative_slope <= 1.0 and f % 4 == 0 and hl > 0 and (hl & (hl - 1)) == 0


def _edge_hubs(lib, csr: CSRGraph, wh_ptr: int, ld_wh: int, n_table: int, slices: int,
               pp: PackedParams, p_sd: int, heads: int, f: int, concat: bool,
               negative_slope: float, bias: torch.Tensor, out: torch.Tensor, stream: int) -> None:
    """Edge kernel with the hub rows split (graph.HubPlan): one launch over the
    hub segments (state stored) and the whole rows (output written), then
    gat_edge_merge for the hubs.  Rows walk graph.rotated_col (long rows)."""
    hubs = csr.hubs
    hf4 = (heads * f + 3) // 4 * 4
    nv = hubs.n_vrows
    st = torch.empty(nv * (hf4 + 2 * heads), dtype=torch.float32, device=out.device)
    p_acc = st.data_ptr()
    p_ml = p_acc + 4 * nv * hf4
    n_pos = hubs.sched_row.numel()
    hint = csr.kernel_hint() if hasattr(csr, "kernel_hint") else \
        csr.num_edges // max(csr.num_nodes, 1)
    rc = lib.gat_edge_aggregate_seg(
        hubs.sched_b.data_ptr(), hubs.sched_e.data_ptr(), 1, rotated_col(csr).data_ptr(),
        hubs.sched_row.data_ptr(), 0, n_pos, wh_ptr, ld_wh, n_table, slices,
        pp.a_src.data_ptr(), pp.c_src.data_ptr(), p_sd, heads, f, int(concat),
        float(negative_slope), p_acc, p_ml, 0, nv, bias.data_ptr(), out.data_ptr(), hint, stream)
    if rc:
        _lib.check(rc, "gat_edge_aggregate_seg (hub split)")
    slot = 0 if hubs.seg_slot is None else hubs.seg_slot.data_ptr()
    rc = lib.gat_edge_merge_ex(hubs.hub_rows.data_ptr(), hubs.hub_vptr.data_ptr(), slot,
                               hubs.n_hub, p_acc, p_ml, heads, f, int(concat), bias.data_ptr(),
                               out.data_ptr(), 0, 0, stream)
    if rc:
        _lib.check(rc, "gat_edge_merge")


class ForwardPlan:
    """The eval forward's launch plan for one (x, graph, layer shape): the
    workspace (Wh | s_src | s_dst), the table layout and the edge path.
    ``gat_forward`` builds one per call; ``bench.py`` keeps one to time the
    two phases of exactly the path the layer runs.

    ``pingpong``: two workspaces, used by alternate ``run()`` calls.  A kernel
    that writes lines the previous kernel gathered from pays for it on this
    GPU (tools/proj_floor.hip: an 11.5-MB streaming write behind a kernel that
    read those lines takes 12.0 us instead of 4.3; the PPI projection 13.8 us
    instead of 10.0), so a layer applied back to back (the layer's cached plan)
    projects into the table the previous forward did NOT read."""

    __slots__ = ("n", "fin", "heads", "f", "hf", "hfp", "concat", "slope", "slices", "split",
                 "ws", "p_wh", "p_ss", "p_sd", "dev", "hint", "khint", "sched", "_csr", "bound",
                 "bufs", "cur", "pws", "need_ss")

    def __init__(self, x: torch.Tensor, csr: CSRGraph, heads: int, f: int, concat: bool,
                 negative_slope: float, pingpong: bool = False):
        n, fin = x.shape
        self.n, self.fin, self.heads, self.f, self.concat = n, fin, heads, f, concat
        self.slope = float(negative_slope)
        self.hf = heads * f
        self.hfp = (self.hf + 3) // 4 * 4
        per = n * (self.hfp + 2 * heads)
        # each workspace starts on a 256-B boundary (the kernels' row alignment)
        per_al = (per + 63) // 64 * 64
        nbuf = 2 if pingpong else 1
        self.ws = torch.empty(per_al * nbuf, dtype=torch.float32, device=x.device)
        self.bufs = []
        for i in range(nbuf):
            p_wh = self.ws.data_ptr() + 4 * per_al * i
            p_ss = p_wh + 4 * n * self.hfp
            self.bufs.append((p_wh, p_ss, p_ss + 4 * n * heads))
        self.cur = 0
        self.p_wh, self.p_ss, self.p_sd = self.bufs[0]
        # the projection's optional workspace (Fin > 128: W split into bf16
        # planes once per call; gat_project_ex), or None
        self.pws = project_workspace(x.device, fin, heads, f)
        self.dev = x.device.index
        self.hint = csr.num_edges // max(n, 1)
        self.slices = wh_slices(heads, f, concat, negative_slope, self.hint)
        # the kernels' hint: + GAT_HINT_LOCAL for a local graph (CSRGraph.kernel_hint)
        self.khint = csr.kernel_hint() if hasattr(csr, "kernel_hint") else self.hint
        self.split = csr.hubs is not None and fused_score_ok(heads, f, negative_slope)
        # short rows: the edge kernel walks a scheduled copy of the CSR (graph.SchedCSR)
        self.sched = None
        if (not self.split and fused_score_ok(heads, f, negative_slope)
                and isinstance(csr, CSRGraph)):
            self.sched = sched_csr(csr)
        # weak: a plan the layer caches must not keep a graph the caller dropped
        # alive (CSRGraph is a tuple, so the weak reference is to its rowptr)
        self._csr = weakref.ref(csr.rowptr)
        self.bound = None  # (pp, bias, lib, project call, edge call) for run()
        # the s_src table: only the gathered-score edge kernels read it (score
        # activations other than LeakyReLU in [0, 1], heads whose F/4 is not a
        # power of two); the fused kernels recompute s_src from the Wh row they
        # gather, so the projection skips it (arxiv: 5.4 MB of stores; layer
        # 85.6 -> 81.3 us, profiles/r05/edge_ab_projss_arxiv.json)
        self.need_ss = not fused_score_ok(heads, f, negative_slope)

    def built_for(self, csr) -> bool:
        """This plan was built for `csr` (and that graph is still alive)."""
        return self._csr() is csr.rowptr

    def run(self, lib, x: torch.Tensor, pp: PackedParams, bias: torch.Tensor,
            out: torch.Tensor, csr: CSRGraph) -> torch.Tensor:
        """project() + edge() for a plan the layer caches between forwards: the
        argument lists (everything but x, out and the stream) are bound once
        per (parameters, bias), so a forward costs two C-ABI calls and little
        Python.  Safe to reuse the workspace: calls on one stream run in order,
        and the layer keys its cached plans by stream."""
        if not self.built_for(csr):
            raise ValueError("ForwardPlan.run: called with a graph the plan was not built for")
        if len(self.bufs) > 1:  # alternate workspaces (pingpong)
            self.cur ^= 1
            self.p_wh, self.p_ss, self.p_sd = self.bufs[self.cur]
        b = self.bound
        if b is None or b[0] is not pp or b[1] != bias.data_ptr() or b[2] is not lib or \
                self.split or self.slices == 1 and b[5]:
            if self.split or self.sched is None:
                self.project(lib, x, pp)
                return self.edge(lib, csr, pp, bias, out)
            b = self.bound = self._bind(lib, pp, bias, csr)
        stream = torch._C._cuda_getCurrentRawStream(self.dev)
        # projection + edge kernel in one C-ABI call (gat_layer_forward)
        rc = b[3](x.data_ptr(), *b[4][self.cur], out.data_ptr(), self.khint, stream)
        if rc:
            if rc == _lib.GAT_EUNSUPPORTED and self.slices > 1:
                # the sliced projection launched nothing: fall back to the
                # row-major table (project() decides)
                self.bound = None
                self.project(lib, x, pp)
                return self.edge(lib, csr, pp, bias, out)
            _lib.check(rc, "gat_layer_forward")
        return out

    def _bind(self, lib, pp: PackedParams, bias: torch.Tensor, csr: CSRGraph):
        n, fin, heads, f, sc = self.n, self.fin, self.heads, self.f, self.sched
        pw = (pp.w.data_ptr(), pp.b.data_ptr(), pp.a_src.data_ptr(), pp.c_src.data_ptr(),
              pp.a_dst.data_ptr(), pp.c_dst.data_ptr())
        p_order = 0 if csr.order is None else csr.order.data_ptr()
        fargs = []
        for p_wh, p_ss, p_sd in self.bufs:  # one argument list per workspace
            fargs.append((n, fin, *pw, heads, f, self.slices, p_wh,
                          p_ss if self.need_ss else 0, p_sd, sc.b.data_ptr(),
                          sc.e.data_ptr(), sc.col.data_ptr(), p_order, int(self.concat),
                          self.slope, bias.data_ptr()))
        return (pp, bias.data_ptr(), lib, lib.gat_layer_forward, fargs, self.slices > 1)

    def project(self, lib, x: torch.Tensor, pp: PackedParams) -> None:
        """gat_project(_sliced / _ex) into the workspace (GAT.py:42-52)."""
        n, fin, heads, f = self.n, self.fin, self.heads, self.f
        stream = torch._C._cuda_getCurrentRawStream(self.dev)  # the current stream, per call
        if self.pws is not None:
            ld = n if self.slices > 1 else self.hfp
            # the sliced edge kernel recomputes s_src from the gathered row:
            # no s_src table then (as gat_project_sliced below)
            p_ss = self.p_ss if self.slices == 1 and self.need_ss else 0
            rc = lib.gat_project_ex(x.data_ptr(), n, fin, pp.w.data_ptr(), pp.b.data_ptr(),
                                    pp.a_src.data_ptr(), pp.c_src.data_ptr(),
                                    pp.a_dst.data_ptr(), pp.c_dst.data_ptr(), heads, f,
                                    self.slices, self.p_wh, ld, p_ss, heads, self.p_sd, 0, 0,
                                    self.pws.data_ptr(), self.pws.numel(), stream)
            if rc == 0:
                return
            if rc != _lib.GAT_EUNSUPPORTED or self.slices == 1:
                _lib.check(rc, "gat_project_ex")
            self.slices = 1  # nothing was launched: the row-major table instead
        if self.slices > 1:
            rc = lib.gat_project_sliced(x.data_ptr(), n, fin, pp.w.data_ptr(), pp.b.data_ptr(),
                                        pp.a_src.data_ptr(), pp.c_src.data_ptr(),
                                        pp.a_dst.data_ptr(), pp.c_dst.data_ptr(), heads, f,
                                        self.slices, self.p_wh, n, 0, heads, self.p_sd,
                                        stream)
            if rc == 0:
                return
            if rc != _lib.GAT_EUNSUPPORTED:
                _lib.check(rc, "gat_project_sliced")
            self.slices = 1  # nothing was launched: the row-major table instead
        rc = lib.gat_project(x.data_ptr(), n, fin, pp.w.data_ptr(), pp.b.data_ptr(),
                             pp.a_src.data_ptr(), pp.c_src.data_ptr(), pp.a_dst.data_ptr(),
                             pp.c_dst.data_ptr(), heads, f, self.p_wh, self.hfp,
                             self.p_ss if self.need_ss else 0,
                             heads, self.p_sd, stream)
        if rc:
            _lib.check(rc, "gat_project")

    def edge(self, lib, csr: CSRGraph, pp: PackedParams, bias: torch.Tensor,
             out: torch.Tensor) -> torch.Tensor:
        """The edge kernel(s) over the table project() wrote (GAT.py:53-67, +bias).
        Short rows walk the scheduled copy (graph.sched_csr), long rows the
        rotated col array (graph.rotated_col): the same edges per row."""
        n, heads, f = self.n, self.heads, self.f
        stream = torch._C._cuda_getCurrentRawStream(self.dev)
        if self.split:
            ld = self.hf // self.slices if self.slices > 1 else self.hfp
            _edge_hubs(lib, csr, self.p_wh, ld, n, self.slices, pp, self.p_sd, heads, f,
                       self.concat, self.slope, bias, out, stream)
            return out
        p_order = 0 if csr.order is None else csr.order.data_ptr()
        sc = self.sched
        if sc is not None:
            ld = self.hf // self.slices if self.slices > 1 else self.hfp
            rc = lib.gat_edge_aggregate_seg(
                sc.b.data_ptr(), sc.e.data_ptr(), 1, sc.col.data_ptr(), p_order, 0, n, self.p_wh,
                ld, n, self.slices, pp.a_src.data_ptr(), pp.c_src.data_ptr(), self.p_sd, heads, f,
                int(self.concat), self.slope, 0, 0, 0, 0, bias.data_ptr(), out.data_ptr(),
                self.khint, stream)
            if rc:
                _lib.check(rc, "gat_edge_aggregate_seg (scheduled CSR)")
            return out
        if self.slices > 1:
            rc = lib.gat_edge_aggregate_sliced(
                csr.rowptr.data_ptr(), rotated_col(csr).data_ptr(), p_order, 0, n, self.p_wh, n,
                self.slices, pp.a_src.data_ptr(), pp.c_src.data_ptr(), self.p_sd, heads, f,
                self.slope, bias.data_ptr(), out.data_ptr(), self.khint, stream)
            if rc:
                _lib.check(rc, "gat_edge_aggregate_sliced")
            return out
        rc = lib.gat_edge_aggregate(
            csr.rowptr.data_ptr(), rotated_col(csr).data_ptr(), p_order, 0, n, self.p_wh, self.hfp,
            self.p_ss if self.need_ss else 0, heads, pp.a_src.data_ptr(), pp.c_src.data_ptr(),
            self.p_sd, heads, f,
            int(self.concat), self.slope, bias.data_ptr(), out.data_ptr(), 0, self.khint, stream)
        if rc:
            _lib.check(rc, "gat_edge_aggregate")
        return out

    def kernel_name(self) -> str:
        if self.sched is not None:
            return (f"gat_edge_aggregate_seg (k_edge_grp over the scheduled CSR"
                    + (f", {self.slices} column planes)" if self.slices > 1 else ")"))
        if self.split:
            return "gat_edge_aggregate_seg (k_edge_grp, hub rows split) + gat_edge_merge"
        if self.slices > 1:
            return f"gat_edge_aggregate_sliced (k_edge_grp, {self.slices} column planes)"
        return "gat_edge_aggregate (k_edge_grp)"


def gat_forward(x: torch.Tensor, csr: CSRGraph, pp: PackedParams, bias: torch.Tensor,
                heads: int, f: int, concat: bool, negative_slope: float = 0.2) -> torch.Tensor:
    """Layer forward on prepared inputs: projection + edge kernel (2 launches;
    3 when hub rows are split).

    Lean host path (it is on the critical path for graphs the size of PPI,
    where the GPU work is ~50 us): one workspace allocation holding
    Wh | s_src | s_dst, one output allocation, two C-ABI calls.  With
    ``wh_slices(...) > 1`` Wh is stored as column planes (``gat_amd.h``,
    sliced node table) and the edge kernel runs one plane per workgroup."""
    lib = _lib.load()
    plan = ForwardPlan(x, csr, heads, f, concat, negative_slope)
    out = torch.empty(plan.n, plan.hf if concat else f, dtype=torch.float32, device=x.device)
    plan.project(lib, x, pp)
    return plan.edge(lib, csr, pp, bias, out)


def score_activation_code(module) -> Tuple[int, float]:
    """Map the layer's ``attention_relu`` module to the library's score
    activation (``GAT_ACT_*``, parameter).  The reference uses
    ``LeakyReLU(0.2)`` (``GAT.py:30``); its activation experiment swaps in
    ``LogSigmoid``, ``Tanh`` and ``Softmax()`` (``run_act_func_experiment.py:111``),
    the last with torch's implicit ``dim=1`` on the 2-D ``[E', H]`` scores."""
    if isinstance(module, torch.nn.LeakyReLU):
        return _lib.GAT_ACT_LEAKY_RELU, float(module.negative_slope)
    if isinstance(module, torch.nn.ReLU):
        return _lib.GAT_ACT_LEAKY_RELU, 0.0
    if isinstance(module, torch.nn.Identity):
        return _lib.GAT_ACT_LEAKY_RELU, 1.0
    if isinstance(module, torch.nn.LogSigmoid):
        return _lib.GAT_ACT_LOG_SIGMOID, 0.0
    if isinstance(module, torch.nn.Tanh):
        return _lib.GAT_ACT_TANH, 0.0
    if isinstance(module, torch.nn.Softmax):
        if module.dim in (None, 1, -1):
            return _lib.GAT_ACT_HEAD_SOFTMAX, 0.0
        raise NotImplementedError(
            f"Softmax(dim={module.dim}) over the edge scores is not supported (dim=1: across heads)")
    raise NotImplementedError(
        f"score activation {type(module).__name__} is not supported by the HIP kernels "
        "(LeakyReLU, ReLU, Identity, LogSigmoid, Tanh, Softmax(dim=1))")


def _check_x(x: torch.Tensor, in_channels: int) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"x must be a torch.Tensor, got {type(x).__name__}")
    if x.device.type != "cuda":
        raise RuntimeError("GraphAttentionLayer runs on a ROCm GPU (MI355X); x is on "
                           f"{x.device}.  There is no CPU path.")
    if x.dim() != 2 or x.size(1) != in_channels:
        raise ValueError(f"x must have shape [N, {in_channels}], got {tuple(x.shape)}")
    if x.dtype != torch.float32:
        raise ValueError(f"x must be float32 (the reference's dtype), got {x.dtype}")
    return x.contiguous()


# layer -> OrderedDict of its cached eval ForwardPlans (GraphAttentionLayer._eval_forward)
_eval_plans: "weakref.WeakKeyDictionary" = weakref.WeakKeyDictionary()


class GraphAttentionLayer(torch.nn.Module):
    """MI355X-native drop-in for the reference ``GraphAttentionLayer``
    (``GAT.py:6``): ``__init__(input_channels, output_channels, num_heads=1,
    concat=False, dropout=0.6)`` and ``forward(x, edge_index)``."""

    def __init__(self, input_channels, output_channels, num_heads=1, concat=False, dropout=0.6):
        super().__init__()
        # PyG MessagePassing(aggr='add', node_dim=0) attributes (GAT.py:9)
        self.aggr = "add"
        self.node_dim = 0
        self.input_channels = input_channels
        self.output_channels = output_channels
        self.num_heads = num_heads
        self.dropout_val = dropout
        # Same module tree and RNG consumption order as GAT.py:16-28, so a
        # seeded construction draws identical parameters.
        self.ws = torch.nn.ModuleList()
        self.attentions1 = torch.nn.ModuleList()
        self.attentions2 = torch.nn.ModuleList()
        for _ in range(num_heads):
            proj = torch.nn.Linear(input_channels, output_channels)
            att_src = torch.nn.Linear(output_channels, 1)
            att_dst = torch.nn.Linear(output_channels, 1)
            for m in (proj, att_src, att_dst):
                torch.nn.init.xavier_uniform_(m.weight)
            self.ws.append(proj)
            self.attentions1.append(att_src)
            self.attentions2.append(att_dst)
        self.attention_relu = torch.nn.LeakyReLU(negative_slope=0.2)
        self.concat = concat
        width = output_channels * num_heads if concat else output_channels
        self.bias = torch.nn.Parameter(torch.zeros(width))
        self._packed: Optional[PackedParams] = None
        self._bind_packed()

    @property
    def negative_slope(self) -> float:
        return float(self.attention_relu.negative_slope)

    def score_activation(self) -> Tuple[int, float]:
        """(GAT_ACT_*, parameter) of ``self.attention_relu`` (read per call, so
        replacing the module after construction takes effect as in the reference)."""
        return score_activation_code(self.attention_relu)

    def _bind_packed(self) -> PackedParams:
        """Make the 6H per-head parameters views into six packed buffers — W
        [H*F, Fin], b, a_src, a_dst [H*F], c_src, c_dst [H] — the layout the
        kernels read, so no forward concatenates parameters and the backward
        returns views of packed gradients.  Values, shapes, dtypes and the
        state_dict are unchanged; optimizers update the views in place."""
        params = _param_list(self)
        H, F = self.num_heads, self.output_channels
        with torch.no_grad():
            w = torch.cat([p.detach().reshape(F, -1) for p in params[0:H]], 0).contiguous()
            flat = [torch.cat([p.detach().reshape(-1) for p in params[k * H:(k + 1) * H]])
                    .contiguous() for k in range(1, 6)]
        b, a_src, c_src, a_dst, c_dst = flat
        for h in range(H):
            params[h].data = w[h * F:(h + 1) * F]
            params[H + h].data = b[h * F:(h + 1) * F]
            params[2 * H + h].data = a_src[h * F:(h + 1) * F].view(1, F)
            params[3 * H + h].data = c_src[h:h + 1]
            params[4 * H + h].data = a_dst[h * F:(h + 1) * F].view(1, F)
            params[5 * H + h].data = c_dst[h:h + 1]
        self._packed = PackedParams(w, b, a_src, c_src, a_dst, c_dst,
                                    tuple(p.data_ptr() for p in params))
        token = self.__dict__.get("_gat_token")
        if token is None or _owners.get(token) is not self:
            token = next(_tokens)
            self.__dict__["_gat_token"] = token
            _owners[token] = self
        for mods in (self.ws, self.attentions1, self.attentions2):
            for m in mods._modules.values():
                m.__dict__["_gat_owner"] = token
        self.__dict__["_packed_dirty"] = False
        return self._packed

    def _packed_aliases(self, pp: PackedParams) -> bool:
        """Head 0's six parameters still start the six packed buffers (their
        pointers at binding time are pp.key[0], [H], [2H] ... [5H]: the packed
        buffers' own pointers, read once instead of on every forward)."""
        mods = self._modules
        if not mods["ws"]._modules:
            return True
        p0 = mods["ws"]._modules["0"]._parameters
        p1 = mods["attentions1"]._modules["0"]._parameters
        p2 = mods["attentions2"]._modules["0"]._parameters
        k, h = pp.key, self.num_heads
        if len(k) != 6 * h:  # (not a _bind_packed key: compare the buffers themselves)
            k = [pp.w.data_ptr()] * h + [pp.b.data_ptr()] * h + [pp.a_src.data_ptr()] * h + \
                [pp.c_src.data_ptr()] * h + [pp.a_dst.data_ptr()] * h + [pp.c_dst.data_ptr()] * h
        return (p0["weight"].data_ptr() == k[0]
                and p0["bias"].data_ptr() == k[h]
                and p1["weight"].data_ptr() == k[2 * h]
                and p1["bias"].data_ptr() == k[3 * h]
                and p2["weight"].data_ptr() == k[4 * h]
                and p2["bias"].data_ptr() == k[5 * h])

    def _apply(self, fn, recurse=True):
        # .to() / .cuda() / .float() replace each parameter's storage: re-pack
        out = super()._apply(fn, recurse)
        self._bind_packed()
        return out

    def packed(self) -> PackedParams:
        """The packed parameter buffers, re-bound if a parameter was replaced
        (registration hook) or re-stored (head 0 no longer aliases them).  A
        ``.data`` reassignment of a later head's parameter is not detected:
        call ``_bind_packed()`` after one."""
        pp = self._packed
        if pp is None or self.__dict__.get("_packed_dirty", True) or \
                not self._packed_aliases(pp):
            pp = self._bind_packed()
        if pp.w.dtype != torch.float32:
            raise ValueError(f"parameters must be float32 (the reference's dtype), got {pp.w.dtype}")
        return pp

    def forward(self, x, edge_index):
        if forward_ad._current_level >= 0:  # inside a dual_level(): elsewhere there are none
            refuse_tangents("GraphAttentionLayer", x, *self.parameters())
        refuse_recording("GraphAttentionLayer")
        x = _check_x(x, self.input_channels)
        csr = get_csr(edge_index, x.size(0), x.device)
        p = float(self.dropout_val) if self.training else 0.0
        needs_grad = torch.is_grad_enabled() and (
            x.requires_grad or any(p_.requires_grad for p_ in self.parameters()))
        act, act_param = self.score_activation()
        default_act = act == _lib.GAT_ACT_LEAKY_RELU and 0.0 <= act_param <= 1.0
        if needs_grad or p > 0.0 or not default_act:
            # training path (training.py): dropout of GAT.py:61 and the HIP backward
            from .training import gat_train_forward, next_seed_slot
            slot = next_seed_slot(self, x.device) if p > 0.0 else None
            return gat_train_forward(self, x, csr, p, 0, act, act_param, seed_slot=slot)
        refuse_recording("GraphAttentionLayer without gradients", jit=True)
        return self._eval_forward(x, csr, act_param)

    def _eval_forward(self, x: torch.Tensor, csr: CSRGraph, slope: float) -> torch.Tensor:
        """The eval forward (GAT.py:37-67, no autograd, no dropout) through a
        ForwardPlan cached per (graph, x shape, slope, stream): its workspace
        and bound argument lists are reused, so a forward allocates only its
        output.  Small graphs (the CIFAR batch: ~15 us of GPU work) are
        host-bound, and this path is most of their host cost."""
        # The plans live in a side table keyed weakly by the layer, not in the
        # module's __dict__: a deepcopy or pickle of the layer must not carry
        # workspaces, raw device pointers or ctypes function pointers along.
        plans = _eval_plans.get(self)
        if plans is None:
            plans = _eval_plans[self] = collections.OrderedDict()
        for k in [k for k, p in plans.items() if p._csr() is None]:  # graphs since freed
            del plans[k]
        dev = x.device.index
        key = (id(csr), x.shape[0], x.shape[1], slope, dev,
               torch._C._cuda_getCurrentRawStream(dev), tuning.generation)
        plan = plans.get(key)
        if plan is None or not plan.built_for(csr):
            plan = plans[key] = ForwardPlan(x, csr, self.num_heads, self.output_channels,
                                            self.concat, slope, pingpong=True)
            while len(plans) > 4:
                plans.popitem(last=False)
        out = torch.empty(plan.n, plan.hf if self.concat else self.output_channels,
                          dtype=torch.float32, device=x.device)
        # (the plan reads only the bias' device pointer: no detached view needed;
        # this path runs without autograd)
        return plan.run(_lib.load(), x, self.packed(), self.bias, out, csr)

    def extra_repr(self) -> str:
        return (f"{self.input_channels}, {self.output_channels}, num_heads={self.num_heads}, "
                f"concat={self.concat}, dropout={self.dropout_val}")


class GraphAttentionLayerActivationTest(GraphAttentionLayer):
    """Counterpart of ``run_act_func_experiment.py:13``: the same layer with the
    score activation passed in (``activation_function``, default LeakyReLU(0.2)).
    Supported: LeakyReLU, ReLU, Identity, LogSigmoid, Tanh, Softmax(dim=1)."""

    def __init__(self, input_channels, output_channels, num_heads=1, concat=False, dropout=0.6,
                 activation_function=None):
        super().__init__(input_channels, output_channels, num_heads=num_heads, concat=concat,
                         dropout=dropout)
        if activation_function is None:
            activation_function = torch.nn.LeakyReLU(negative_slope=0.2)
        score_activation_code(activation_function)  # fail at construction if unsupported
        self.attention_relu = activation_function
