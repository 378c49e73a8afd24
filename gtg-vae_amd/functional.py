"""torch.autograd.Function wrappers over the C ABI (include/gtgvae.h).

PyTorch is used for device memory, streams and the autograd graph only; every
arithmetic step of forward and backward runs in csrc/*.hip.  All tensors must
be on the GPU, and fp32 but for the operators on rows of vocabulary logits, which
take fp32, fp16 and bf16 logits; there is no fallback.
"""
import functools
from typing import Optional

import torch

from . import _lib
from ._lib import check, ptr, stream_ptr


def _on_tensor_device(fn):
    """Run ``fn`` with the device of its first GPU tensor argument current, so that the stream handed to the
    library (the current stream) and the kernels' launch device are the tensors' device even when the caller's
    current device is another GPU."""
    @functools.wraps(fn)
    def wrapped(*args, **kwargs):
        for a in args:
            if isinstance(a, torch.Tensor) and a.is_cuda:
                if a.device.index == torch.cuda.current_device():
                    break
                with torch.cuda.device(a.device):
                    return fn(*args, **kwargs)
        return fn(*args, **kwargs)
    return wrapped


def _f32c(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None:
        return None
    _lib.require_cuda(t)
    if t.dtype != torch.float32:
        t = t.float()
    return t.contiguous()


def _ws(nbytes: int, device) -> torch.Tensor:
    return torch.empty((max(int(nbytes), 256),), dtype=torch.uint8, device=device)


# ---------------------------------------------------------------------------
# adjacency
# ---------------------------------------------------------------------------
@_on_tensor_device
def build_adj(edge_index: torch.Tensor, num_graphs: int, nmax: int, check_edges: bool = False,
              return_extents: bool = False):
    """D^-1/2 (C + I) D^-1/2 per graph, (B, nmax, nmax) fp32, from a PyG-style
    batched edge_index (2, E) int64.  With check_edges the error flag is read
    back (a host sync) and an exception raised if an edge leaves its graph.
    With return_extents the per-graph extents (B) int32 are returned as well
    (1 + the highest node index an edge touches: the rows the compact encoder
    stores; EncoderFn's ``extents`` argument)."""
    _lib.require_cuda(edge_index)
    ei = edge_index.contiguous()
    if ei.dtype != torch.int64:
        ei = ei.long()
    dev = ei.device
    counts = torch.zeros((num_graphs * nmax * nmax,), dtype=torch.int32, device=dev)  # zero in, zero out
    err = torch.zeros((1,), dtype=torch.int32, device=dev)
    adj = torch.empty((num_graphs, nmax, nmax), dtype=torch.float32, device=dev)
    extents = torch.empty((num_graphs,), dtype=torch.int32, device=dev)
    check(_lib.lib().gtg_adj_build(ptr(ei), ei.shape[1], num_graphs, nmax, ptr(counts), ptr(err), ptr(adj),
                                   ptr(extents), stream_ptr()), "gtg_adj_build")
    if check_edges and int(err.item()) != 0:
        raise _lib.GtgError("edge_index holds an edge whose endpoints are out of range or in different graphs")
    return (adj, extents) if return_extents else adj


# ---------------------------------------------------------------------------
# encoder
# ---------------------------------------------------------------------------
class EncoderFn(torch.autograd.Function):
    """pooled (B, d) = global_max_pool(GCN2(relu(GCN1(x))))."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, adj, x, W1, b1, W2, b2, extents=None, matrix_mode=None):
        L = _lib.lib()
        ctx.mode = mode = _lib.matrix_mode(matrix_mode)
        adj, x, W1, b1, W2, b2 = map(_f32c, (adj, x, W1, b1, W2, b2))
        B, n, _ = adj.shape
        H, f = W1.shape
        d = W2.shape[0]
        if H != 2 * d or W2.shape[1] != H:
            raise _lib.GtgError("encoder weights must be W1 (2d, f), W2 (d, 2d)")
        if x is not None and tuple(x.shape) != (B * n, f):
            raise _lib.GtgError(f"x must be (B*n, f) = ({B * n}, {f}), got {tuple(x.shape)}")
        dev = adj.device
        ctx.compact = x is None and extents is not None and f == n
        if ctx.compact:
            # identity features: only the rows an edge touches are stored and multiplied
            meta = torch.empty((2 * B + 2,), dtype=torch.int32, device=dev)
            adjc = torch.empty((B * n + n, n), dtype=torch.float32, device=dev)
            h1c = torch.empty((B * n + n, H), dtype=torch.float32, device=dev)
            pooled = torch.empty((B, d), dtype=torch.float32, device=dev)
            argmax = torch.empty((B, d), dtype=torch.int32, device=dev)
            ws = _ws(L.gtg_encoder_compact_fwd_workspace_bytes(B, n, d), dev)
            check(L.gtg_encoder_compact_fwd(ptr(adj), ptr(extents), ptr(W1), ptr(b1), ptr(W2), ptr(b2), B, n, d,
                                            ptr(meta), ptr(adjc), ptr(h1c), ptr(pooled), ptr(argmax), mode, ptr(ws),
                                            ws.numel(), stream_ptr()), "gtg_encoder_compact_fwd")
            ctx.save_for_backward(adj, adjc, meta, W2, h1c, argmax)
            ctx.dims = (B, n, f, d)
            ctx.mark_non_differentiable(argmax)
            return pooled, argmax
        h1 = torch.empty((B * n, H), dtype=torch.float32, device=dev)
        pooled = torch.empty((B, d), dtype=torch.float32, device=dev)
        argmax = torch.empty((B, d), dtype=torch.int32, device=dev)
        nb = L.gtg_encoder_fwd_workspace_bytes(B, n, f, d, int(x is not None))
        ws = _ws(nb, dev)
        check(L.gtg_encoder_fwd(ptr(adj), ptr(x), ptr(W1), ptr(b1), ptr(W2), ptr(b2), B, n, f, d, ptr(h1), ptr(pooled),
                                ptr(argmax), mode, ptr(ws), ws.numel(), stream_ptr()), "gtg_encoder_fwd")
        ctx.save_for_backward(adj, x, W1, W2, h1, argmax)
        ctx.dims = (B, n, f, d)
        ctx.mark_non_differentiable(argmax)
        return pooled, argmax

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dpooled, _dargmax):
        L = _lib.lib()
        B, n, f, d = ctx.dims
        dpooled = _f32c(dpooled)
        dev = dpooled.device
        dW1 = torch.empty((2 * d, f), dtype=torch.float32, device=dev)
        db1 = torch.empty((2 * d,), dtype=torch.float32, device=dev)
        dW2 = torch.empty((d, 2 * d), dtype=torch.float32, device=dev)
        db2 = torch.empty((d,), dtype=torch.float32, device=dev)
        if ctx.compact:
            adj, adjc, meta, W2, h1c, argmax = ctx.saved_tensors
            ws = _ws(L.gtg_encoder_compact_bwd_workspace_bytes(B, n, d), dev)
            check(L.gtg_encoder_compact_bwd(ptr(adj), ptr(adjc), ptr(meta), ptr(W2), ptr(h1c), ptr(argmax),
                                            ptr(dpooled), B, n, d, ptr(dW1), ptr(db1), ptr(dW2), ptr(db2), ctx.mode,
                                            ptr(ws), ws.numel(), stream_ptr()), "gtg_encoder_compact_bwd")
            return None, None, dW1, db1, dW2, db2, None, None
        adj, x, W1, W2, h1, argmax = ctx.saved_tensors
        nb = L.gtg_encoder_bwd_workspace_bytes(B, n, f, d, int(x is not None))
        ws = _ws(nb, dev)
        check(L.gtg_encoder_bwd(ptr(adj), ptr(x), ptr(W1), ptr(W2), ptr(h1), ptr(argmax), ptr(dpooled), B, n, f, d,
                                ptr(dW1), ptr(db1), ptr(dW2), ptr(db2), ctx.mode, ptr(ws), ws.numel(), stream_ptr()),
              "gtg_encoder_bwd")
        # node features and the adjacency are inputs, not parameters: no gradient
        return None, None, dW1, db1, dW2, db2, None, None


# ---------------------------------------------------------------------------
# latent head
# ---------------------------------------------------------------------------
class LatentFn(torch.autograd.Function):
    """(z, kl, mu, logvar) from h with eps supplied; mu/logvar are returned for
    inspection only (non-differentiable outputs)."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, h, Wmu, bmu, Wlv, blv, eps):
        L = _lib.lib()
        h, Wmu, bmu, Wlv, blv, eps = map(_f32c, (h, Wmu, bmu, Wlv, blv, eps))
        B, d = h.shape
        dev = h.device
        mu = torch.empty((B, d), dtype=torch.float32, device=dev)
        lv = torch.empty_like(mu)
        z = torch.empty_like(mu)
        kl = torch.empty((), dtype=torch.float32, device=dev)
        ws = _ws(L.gtg_latent_workspace_bytes(B, d), dev)
        check(L.gtg_latent_fwd(ptr(h), ptr(Wmu), ptr(bmu), ptr(Wlv), ptr(blv), ptr(eps), B, d, ptr(mu), ptr(lv), ptr(z),
                               ptr(kl), ptr(ws), ws.numel(), stream_ptr()), "gtg_latent_fwd")
        ctx.save_for_backward(h, Wmu, Wlv, mu, lv, eps)
        ctx.mark_non_differentiable(mu, lv)
        return z, kl, mu, lv

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dz, dkl, _dmu, _dlv):
        L = _lib.lib()
        h, Wmu, Wlv, mu, lv, eps = ctx.saved_tensors
        B, d = h.shape
        dev = h.device
        dz = _f32c(dz)
        dkl = _f32c(dkl) if dkl is not None else None
        dWmu = torch.empty_like(Wmu)
        dWlv = torch.empty_like(Wlv)
        dbmu = torch.empty((d,), dtype=torch.float32, device=dev)
        dblv = torch.empty((d,), dtype=torch.float32, device=dev)
        dh = torch.empty_like(h)
        ws = _ws(L.gtg_latent_workspace_bytes(B, d), dev)
        kl_w = 1.0 if dkl is not None else 0.0
        check(L.gtg_latent_bwd(ptr(h), ptr(Wmu), ptr(Wlv), ptr(mu), ptr(lv), ptr(eps), ptr(dz), kl_w, ptr(dkl), B, d,
                               ptr(dWmu), ptr(dbmu), ptr(dWlv), ptr(dblv), ptr(dh), ptr(ws), ws.numel(), stream_ptr()),
              "gtg_latent_bwd")
        return dh, dWmu, dbmu, dWlv, dblv, None


class ReparamKLFn(torch.autograd.Function):
    """(z, kl) from (mu, logvar, eps): GTVAE.reparameterize + GTVAE.loss_kl."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, mu, logvar, eps):
        L = _lib.lib()
        mu, logvar, eps = map(_f32c, (mu, logvar, eps))
        B, d = mu.shape
        z = torch.empty_like(mu)
        kl = torch.empty((), dtype=torch.float32, device=mu.device)
        ws = _ws(L.gtg_latent_workspace_bytes(B, d), mu.device)
        check(L.gtg_reparam_kl_fwd(ptr(mu), ptr(logvar), ptr(eps), B, d, ptr(z), ptr(kl), ptr(ws), ws.numel(),
                                   stream_ptr()), "gtg_reparam_kl_fwd")
        ctx.save_for_backward(mu, logvar, eps)
        return z, kl

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dz, dkl):
        L = _lib.lib()
        mu, logvar, eps = ctx.saved_tensors
        B, d = mu.shape
        dz = _f32c(dz)
        dkl = _f32c(dkl) if dkl is not None else None
        dmu = torch.empty_like(mu)
        dlv = torch.empty_like(mu)
        check(L.gtg_reparam_kl_bwd(ptr(mu), ptr(logvar), ptr(eps), ptr(dz), 1.0 if dkl is not None else 0.0, ptr(dkl),
                                   B, d, ptr(dmu), ptr(dlv), stream_ptr()), "gtg_reparam_kl_bwd")
        return dmu, dlv, None


# ---------------------------------------------------------------------------
# decoder and reconstruction loss
# ---------------------------------------------------------------------------
class DecoderFn(torch.autograd.Function):
    """out (B, M) = sigmoid(relu(z D1^T + c1) D2^T + c2)."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, z, D1, c1, D2, c2):
        L = _lib.lib()
        z, D1, c1, D2, c2 = map(_f32c, (z, D1, c1, D2, c2))
        B, d = z.shape
        hid = D1.shape[0]
        m_out = D2.shape[0]
        y1 = torch.empty((B, hid), dtype=torch.float32, device=z.device)
        out = torch.empty((B, m_out), dtype=torch.float32, device=z.device)
        check(L.gtg_decoder_fwd(ptr(z), ptr(D1), ptr(c1), ptr(D2), ptr(c2), B, d, hid, m_out, ptr(y1), ptr(out),
                                stream_ptr()), "gtg_decoder_fwd")
        ctx.save_for_backward(z, D1, D2, y1, out)
        return out

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dout):
        L = _lib.lib()
        z, D1, D2, y1, out = ctx.saved_tensors
        B, d = z.shape
        hid, m_out = D1.shape[0], D2.shape[0]
        dev = z.device
        dout = _f32c(dout)
        dD1 = torch.empty_like(D1)
        dD2 = torch.empty_like(D2)
        dc1 = torch.empty((hid,), dtype=torch.float32, device=dev)
        dc2 = torch.empty((m_out,), dtype=torch.float32, device=dev)
        dz = torch.empty_like(z)
        ws = _ws(L.gtg_decoder_bwd_workspace_bytes(B, d, hid, m_out), dev)
        check(L.gtg_decoder_bwd(ptr(z), ptr(D1), ptr(D2), ptr(y1), ptr(out), ptr(dout), None, 0, 1.0, None, B, d, hid,
                                m_out, ptr(dD1), ptr(dc1), ptr(dD2), ptr(dc2), ptr(dz), ptr(ws), ws.numel(),
                                stream_ptr()), "gtg_decoder_bwd")
        return dz, dD1, dc1, dD2, dc2


class BCELossFn(torch.autograd.Function):
    """mean_b mean_k BCE(out[b,k], triu(adj[b])[k]) (log clamped at -100)."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, out, adj):
        L = _lib.lib()
        out, adj = _f32c(out), _f32c(adj)
        B, m = out.shape
        n = adj.shape[-1]
        if tuple(adj.shape) != (B, n, n) or m != n * (n + 1) // 2:
            raise _lib.GtgError(f"out {tuple(out.shape)} / adj {tuple(adj.shape)} do not match (B, n(n+1)/2) / (B, n, n)")
        loss = torch.empty((), dtype=torch.float32, device=out.device)
        ws = _ws(L.gtg_bce_workspace_bytes(B), out.device)
        check(L.gtg_bce_loss_fwd(ptr(out), ptr(adj), B, n, ptr(loss), None, None, ptr(ws), ws.numel(), stream_ptr()),
              "gtg_bce_loss_fwd")
        ctx.save_for_backward(out, adj)
        return loss

    @staticmethod
    @_on_tensor_device
    def backward(ctx, g):
        L = _lib.lib()
        out, adj = ctx.saved_tensors
        B, n = adj.shape[0], adj.shape[-1]
        g = _f32c(g)
        dout = torch.empty_like(out)
        check(L.gtg_bce_loss_bwd(ptr(out), ptr(adj), 1.0, ptr(g), B, n, 0, ptr(dout), stream_ptr()),
              "gtg_bce_loss_bwd")
        return dout, None


@_on_tensor_device
def edge_precision_recall(edges: torch.Tensor, count: torch.Tensor, gold_bits: torch.Tensor, nmax: int):
    """Per-graph (recall, precision) fp32 tensors on the GPU."""
    _lib.require_cuda(edges, count, gold_bits)
    G = count.shape[0]
    rec = torch.empty((G,), dtype=torch.float32, device=edges.device)
    prec = torch.empty_like(rec)
    check(_lib.lib().gtg_edge_prf(ptr(edges.contiguous()), ptr(count.contiguous()), ptr(gold_bits.contiguous()), G,
                                  nmax, ptr(rec), ptr(prec), stream_ptr()), "gtg_edge_prf")
    return rec, prec


@_on_tensor_device
def gemm(A, B, a_kc=True, b_kc=True, bias=None, epilogue=0, aux=None, out=None, M=None, N=None, K=None,
         split_k=True, matrix_mode="f32"):
    """Thin test/profiling hook over gtg_gemm_f32 (see include/gtgvae.h)."""
    L = _lib.lib()
    A, B = _f32c(A), _f32c(B)
    if M is None:
        M, K = (A.shape[0], A.shape[1]) if a_kc else (A.shape[1], A.shape[0])
        N = B.shape[0] if b_kc else B.shape[1]
    C = out if out is not None else torch.empty((M, N), dtype=torch.float32, device=A.device)
    slabs = None
    nb = L.gtg_gemm_splitk_workspace_bytes(M, N, K) if split_k else 0
    if nb:
        slabs = _ws(nb, A.device)
    check(L.gtg_gemm_f32(ptr(A), ptr(B), ptr(C), M, N, K, A.stride(0), B.stride(0), C.stride(0), int(a_kc), int(b_kc),
                         ptr(_f32c(bias)), epilogue, ptr(_f32c(aux)), aux.stride(0) if aux is not None else 0,
                         ptr(slabs), nb, _lib.matrix_mode(matrix_mode), stream_ptr()), "gtg_gemm_f32")
    return C


@_on_tensor_device
def gemm_rows(A, B, a_kc=True, b_kc=True, rows_dev=None, bias=None, epilogue=0, aux=None, out=None, matrix_mode="f32"):
    """Test/profiling hook over gtg_gemm_f32_rows: the GEMM of the compact-row
    encoder (row count read on the device, tail tiles split along K)."""
    L = _lib.lib()
    A, B = _f32c(A), _f32c(B)
    M, K = (A.shape[0], A.shape[1]) if a_kc else (A.shape[1], A.shape[0])
    N = B.shape[0] if b_kc else B.shape[1]
    C = out if out is not None else torch.zeros((M, N), dtype=torch.float32, device=A.device)
    ws = _ws(L.gtg_gemm_rows_workspace_bytes(), A.device)
    check(L.gtg_gemm_f32_rows(ptr(A), ptr(B), ptr(C), M, N, K, A.stride(0), B.stride(0), C.stride(0), int(a_kc),
                              int(b_kc), ptr(_f32c(bias)), epilogue, ptr(_f32c(aux)),
                              aux.stride(0) if aux is not None else 0, ptr(rows_dev), _lib.matrix_mode(matrix_mode),
                              ptr(ws), ws.numel(), stream_ptr()),
          "gtg_gemm_f32_rows")
    return C


@_on_tensor_device
def split_planes(x: torch.Tensor, transpose: bool = False) -> torch.Tensor:
    """k-blocked bf16 planes (3, K/16, R, 16) of the (R, K) operand x -- or of x^T with transpose -- whose sum is
    the operand exactly; K must be a multiple of 16."""
    x = _f32c(x)
    rows, cols = x.shape
    R, K = (cols, rows) if transpose else (rows, cols)
    out = torch.empty((3, K // 16, R, 16), dtype=torch.bfloat16, device=x.device)
    check(_lib.lib().gtg_split_planes(ptr(x), rows, cols, x.stride(0), int(transpose), ptr(out), stream_ptr()),
          "gtg_split_planes")
    return out


@_on_tensor_device
def gemm_planes_rows(Ap, Bp, rows_dev=None, bias=None, epilogue=0, aux=None, out=None):
    """Test/profiling hook over gtg_gemm_planes_rows: C = epilogue(A B^T) from k-blocked planes (split_planes)."""
    L = _lib.lib()
    _, KB, M, _ = Ap.shape
    K, N = KB * 16, Bp.shape[2]
    C = out if out is not None else torch.zeros((M, N), dtype=torch.float32, device=Ap.device)
    ws = _ws(L.gtg_gemm_rows_workspace_bytes(), Ap.device)
    check(L.gtg_gemm_planes_rows(ptr(Ap), ptr(Bp), ptr(C), M, N, K, C.stride(0), ptr(_f32c(bias)), epilogue,
                                 ptr(_f32c(aux)), aux.stride(0) if aux is not None else 0, ptr(rows_dev), ptr(ws),
                                 ws.numel(), stream_ptr()), "gtg_gemm_planes_rows")
    return C


# ---------------------------------------------------------------------------
# weight gradients written where the optimiser reads them
# ---------------------------------------------------------------------------
def _grad_slot(weight, shape) -> Optional[torch.Tensor]:
    """``weight.grad`` when the weight asks for its gradient to be STORED there: its ``grad_overwrite`` attribute
    is true and ``.grad`` is already a dense contiguous fp32 GPU tensor of ``shape`` (JointTrainer's flat gradient
    buffer).  The backward then writes the gradient into that tensor, replacing what it held -- right for a weight
    that one call per backward pass uses, in a buffer nobody accumulates over passes -- and returns None to
    autograd: no temporary, no ``grad += new`` pass over the weight.  (The weight's post-accumulate-grad hooks run
    as usual: autograd calls them for a None gradient too, after the backward that stored it has returned.)"""
    if weight is None or not getattr(weight, "grad_overwrite", False):
        return None
    g = weight.grad
    if g is not None and g.is_cuda and g.dtype == torch.float32 and g.is_contiguous() and tuple(g.shape) == tuple(shape):
        return g
    return None


# ---------------------------------------------------------------------------
# nn.Linear on the library's GEMM (the text branch's small layers)
# ---------------------------------------------------------------------------
class LinearFn(torch.autograd.Function):
    """y (rows, out) = x W^T + b (text_vae.py:41-42 hgen, z2emb): forward, dx = dy W and dW = dy^T x on the fp32
    matrix pipe (the layers are a few hundred MFLOP: the matrix mode's split products would buy nothing); db, the
    column sums of dy, is a torch reduction."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, x, W, b):
        x2, Wc, bc = _f32c(x.reshape(-1, x.shape[-1])), _f32c(W), _f32c(b)
        if Wc.dim() != 2 or Wc.shape[1] != x2.shape[1] or (bc is not None and bc.numel() != Wc.shape[0]):
            raise _lib.GtgError("linear: x (..., in), W (out, in), b (out)")
        y = gemm(x2, Wc, True, True, bias=bc)
        ctx.save_for_backward(x2, Wc)
        ctx.lead = tuple(x.shape[:-1])
        ctx.has_bias = b is not None
        return y.view(ctx.lead + (Wc.shape[0],))

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dy):
        x2, W = ctx.saved_tensors
        dy2 = _f32c(dy.reshape(-1, W.shape[0]))
        dx = gemm(dy2, W, True, False).view(ctx.lead + (W.shape[1],)) if ctx.needs_input_grad[0] else None
        dW = gemm(dy2, x2, False, False) if ctx.needs_input_grad[1] else None
        db = dy2.sum(0) if (ctx.has_bias and ctx.needs_input_grad[2]) else None
        return dx, dW, db


def linear(x, W, b=None):
    """x W^T + b; see LinearFn."""
    return LinearFn.apply(x, W, b)


# ---------------------------------------------------------------------------
# vocabulary projection + token cross-entropy (text decoder)
# ---------------------------------------------------------------------------
class ProjCEFn(torch.autograd.Function):
    """loss (rows) = cross_entropy(H W^T + b, targets, ignore_index=padidx, reduction='none'),
    pred (rows) int32 = argmax of the logits (-1 where the target is the pad symbol).

    text_vae.py:65 (self.proj) + :77-79 (loss_rec) + :83-84 (accuracy's arg-max)
    without ever holding the logits of pad tokens: those rows are left out of
    all three GEMMs."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, H, W, b, targets, padidx, matrix_mode=None):
        L = _lib.lib()
        ctx.mode = mode = _lib.matrix_mode(matrix_mode)
        ctx.w_param = W
        H, W, b = map(_f32c, (H, W, b))
        _lib.require_cuda(targets)
        targets = targets.contiguous().long().view(-1)
        R, K = H.shape
        V = W.shape[0]
        if W.shape[1] != K or targets.numel() != R or (b is not None and b.numel() != V):
            raise _lib.GtgError("proj_ce: H (rows, k), W (vocab, k), b (vocab), targets (rows)")
        dev = H.device
        ldp = (V + 31) // 32 * 32
        loss = torch.empty((R,), dtype=torch.float32, device=dev)
        pred = torch.empty((R,), dtype=torch.int32, device=dev)
        rowmap = torch.empty((2 * R + 1,), dtype=torch.int32, device=dev)
        Hc = torch.empty((R, K), dtype=torch.float32, device=dev)
        P = torch.empty((R, ldp), dtype=torch.float32, device=dev)
        ws = _ws(L.gtg_proj_ce_fwd_workspace_bytes(R, K, V), dev)
        check(L.gtg_proj_ce_fwd(ptr(H), ptr(W), ptr(b), ptr(targets), R, K, V, int(padidx), ptr(loss), ptr(pred),
                                ptr(rowmap), ptr(Hc), ptr(P), ldp, mode, ptr(ws), ws.numel(), stream_ptr()),
              "gtg_proj_ce_fwd")
        ctx.save_for_backward(W, rowmap, Hc, P)
        ctx.dims = (R, K, V, ldp, b is not None)
        ctx.mark_non_differentiable(pred)
        return loss, pred

    @staticmethod
    @_on_tensor_device
    def backward(ctx, gloss, _gpred):
        L = _lib.lib()
        W, rowmap, Hc, P = ctx.saved_tensors
        R, K, V, ldp, has_bias = ctx.dims
        gloss = _f32c(gloss).view(-1)
        dev = gloss.device
        dH = torch.empty((R, K), dtype=torch.float32, device=dev) if ctx.needs_input_grad[0] else None
        slot = _grad_slot(ctx.w_param, (V, K))   # the weight's own .grad, if it asks for that (see _grad_slot)
        dW = slot if slot is not None else torch.empty((V, K), dtype=torch.float32, device=dev)
        db = torch.empty((V,), dtype=torch.float32, device=dev) if has_bias else None
        ws = _ws(L.gtg_proj_ce_bwd_workspace_bytes(R, K, V), dev)
        check(L.gtg_proj_ce_bwd(ptr(W), ptr(gloss), ptr(rowmap), ptr(Hc), ptr(P), ldp, R, K, V, ptr(dH), ptr(dW),
                                ptr(db), ctx.mode, ptr(ws), ws.numel(), stream_ptr()), "gtg_proj_ce_bwd")
        return dH, (None if slot is not None else dW), db, None, None, None


def lstm_applies(T: int, B: int, I: int, H: int) -> bool:
    """Sizes the HIP recurrence takes (include/gtgvae.h, gtg_lstm_fwd)."""
    return T >= 1 and B >= 1 and I >= 4 and I % 4 == 0 and H >= 64 and H % 64 == 0 and T * B * 4 * H < 2 ** 31


class LSTMFn(torch.autograd.Function):
    """One direction of a one-layer nn.LSTM over a padded sequence (text_vae.py:37-40, called at :57 and :64):
    x (T, B, I) -> (every step's hidden state (T, B, H) in time order, h_n (B, H), c_n (B, H)).  ``reverse`` runs
    time backwards (the module's ``*_reverse`` weights); h0 / c0 (B, H) or None."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, x, w_ih, w_hh, b_ih, b_hh, h0, c0, reverse=False, matrix_mode=None):
        L = _lib.lib()
        ctx.mode = mode = _lib.matrix_mode(matrix_mode)
        ctx.w_params = (w_ih, w_hh)
        x, w_ih, w_hh, b_ih, b_hh, h0, c0 = map(_f32c, (x, w_ih, w_hh, b_ih, b_hh, h0, c0))
        T, B, I = x.shape
        H = w_hh.shape[1]
        if w_ih.shape != (4 * H, I) or w_hh.shape != (4 * H, H) or b_ih.numel() != 4 * H or b_hh.numel() != 4 * H or \
                any(t is not None and t.shape != (B, H) for t in (h0, c0)):
            raise _lib.GtgError("lstm: x (T, B, I), w_ih (4H, I), w_hh (4H, H), biases (4H), h0 / c0 (B, H)")
        if not lstm_applies(T, B, I, H):
            raise _lib.GtgError("lstm: the HIP recurrence needs I % 4 == 0 and H % 64 == 0")
        dev = x.device
        hs = torch.empty((T, B, H), dtype=torch.float32, device=dev)
        cs = torch.empty((T, B, H), dtype=torch.float32, device=dev)
        gates = torch.empty((T, B, 4 * H), dtype=torch.float32, device=dev)
        ws = _ws(L.gtg_lstm_fwd_workspace_bytes(T, B, I, H), dev)
        check(L.gtg_lstm_fwd(ptr(x), ptr(w_ih), ptr(w_hh), ptr(b_ih), ptr(b_hh), ptr(h0), ptr(c0), T, B, I, H,
                             int(bool(reverse)), ptr(hs), ptr(cs), ptr(gates), mode, ptr(ws), ws.numel(), stream_ptr()),
              "gtg_lstm_fwd")
        ctx.save_for_backward(x, w_ih, w_hh, h0, c0, hs, cs, gates)
        ctx.dims = (T, B, I, H, bool(reverse))
        # an output nobody differentiates through (the encoder uses h_n alone) reaches backward as None, which
        # gtg_lstm_bwd takes as "no gradient", instead of a (T, B, H) block of zeros read at every time step
        ctx.set_materialize_grads(False)
        last = 0 if reverse else T - 1
        return hs, hs[last].clone(), cs[last].clone()

    @staticmethod
    @_on_tensor_device
    def backward(ctx, d_hs, d_hT, d_cT):
        L = _lib.lib()
        x, w_ih, w_hh, h0, c0, hs, cs, gates = ctx.saved_tensors
        T, B, I, H, reverse = ctx.dims
        d_hs, d_hT, d_cT = map(_f32c, (d_hs, d_hT, d_cT))
        dev = x.device
        need = ctx.needs_input_grad
        dx = torch.empty((T, B, I), dtype=torch.float32, device=dev) if need[0] else None
        s_ih, s_hh = _grad_slot(ctx.w_params[0], (4 * H, I)), _grad_slot(ctx.w_params[1], (4 * H, H))
        dw_ih = s_ih if s_ih is not None else torch.empty((4 * H, I), dtype=torch.float32, device=dev)
        dw_hh = s_hh if s_hh is not None else torch.empty((4 * H, H), dtype=torch.float32, device=dev)
        db = torch.empty((4 * H,), dtype=torch.float32, device=dev)
        dh0 = torch.empty((B, H), dtype=torch.float32, device=dev) if (h0 is not None and need[5]) else None
        dc0 = torch.empty((B, H), dtype=torch.float32, device=dev) if (c0 is not None and need[6]) else None
        ws = _ws(L.gtg_lstm_bwd_workspace_bytes(T, B, I, H), dev)
        check(L.gtg_lstm_bwd(ptr(x), ptr(w_ih), ptr(w_hh), ptr(h0), ptr(c0), ptr(hs), ptr(cs), ptr(gates), ptr(d_hs),
                             ptr(d_hT), ptr(d_cT), T, B, I, H, int(reverse), ptr(dx), ptr(dw_ih), ptr(dw_hh), ptr(db),
                             ptr(dh0), ptr(dc0), ctx.mode, ptr(ws), ws.numel(), stream_ptr()), "gtg_lstm_bwd")
        return (dx, None if s_ih is not None else dw_ih, None if s_hh is not None else dw_hh, db, db, dh0, dc0, None,
                None)


def lstm(x, w_ih, w_hh, b_ih, b_hh, h0=None, c0=None, reverse=False, matrix_mode=None):
    """(hs (T, B, H), h_n (B, H), c_n (B, H)) of one LSTM direction; see LSTMFn."""
    return LSTMFn.apply(x, w_ih, w_hh, b_ih, b_hh, h0, c0, reverse, matrix_mode)


def proj_ce(H, W, b, targets, padidx, matrix_mode=None):
    """Per-token cross-entropy of the projected decoder outputs and the arg-max token; see ProjCEFn."""
    return ProjCEFn.apply(H, W, b, targets, padidx, matrix_mode)


# ---------------------------------------------------------------------------
# text branch: word drop, embedding lookup + dropout, dropout
# ---------------------------------------------------------------------------
def _rng_key():
    """(seed, stream id) for one randomised forward call: the seed is PyTorch's (``torch.manual_seed``), the stream
    id is drawn from PyTorch's default CPU generator -- no device work, no synchronisation, and a run repeats
    under the same ``torch.manual_seed`` exactly as stock dropout does.  The library's keep decisions are a pure
    function of (seed, stream id, element index), so the backward regenerates the forward's mask from this pair."""
    seed = torch.initial_seed() & 0xFFFFFFFFFFFFFFFF
    sid = int(torch.randint(0, 2 ** 62, (1,)).item())
    return seed, sid


@_on_tensor_device
def word_drop(x: torch.Tensor, padidx: int, p: float, keep: Optional[torch.Tensor] = None) -> torch.Tensor:
    """noise.word_drop (noise.py:12-22) on the device: x (T, B) int64 token ids; every token of a column but the
    first is dropped with probability p, the kept ones move up in order, the tail is filled with padidx.
    ``keep`` (T, B) bool / uint8: an explicit keep mask instead of the random one."""
    _lib.require_cuda(x)
    T, B = x.shape
    x = x.contiguous().long()
    out = torch.empty_like(x)
    k = None if keep is None else keep.to(device=x.device, dtype=torch.uint8).contiguous()
    seed, sid = (0, 0) if k is not None else _rng_key()
    check(_lib.lib().gtg_word_drop(ptr(x), T, B, int(padidx), float(p), seed, sid, ptr(k), ptr(out), stream_ptr()),
          "gtg_word_drop")
    return out


class EmbedDropoutFn(torch.autograd.Function):
    """drop(weight[ids]) (+ add broadcast over the leading dimension): text_vae.py:56 and :62 in one kernel, the
    backward an ordered scatter-add.  ids (T, B) int64, weight (V, D), add (B, D) or None -> (T, B, D).

    A weight whose ``grad_inplace`` attribute is true and whose ``.grad`` is already a dense tensor (JointTrainer's
    flat gradient buffer) receives its gradient by accumulation into that tensor -- the backward then returns None
    for it, and no (V, D) temporary is made; otherwise a dense (V, D) gradient is returned to autograd."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, ids, weight, add, p):
        L = _lib.lib()
        _lib.require_cuda(ids, weight, add)
        T, B = ids.shape
        V, D = weight.shape
        if D % 4:
            raise _lib.GtgError("embed_dropout: the embedding width must be a multiple of 4")
        w = _f32c(weight)
        a = _f32c(add)
        if a is not None and tuple(a.shape) != (B, D):
            raise _lib.GtgError("embed_dropout: add must be (B, D)")
        ids_c = ids.contiguous().long()
        out = torch.empty((T, B, D), dtype=torch.float32, device=w.device)
        err = torch.zeros(1, dtype=torch.int32, device=w.device) if EmbedDropoutFn.check_ids else None
        seed, sid = _rng_key() if p > 0 else (0, 0)
        check(L.gtg_embed_dropout_fwd(ptr(w), ptr(ids_c), T * B, V, D, float(p), seed, sid, ptr(a), B if a is not None else 0,
                                      ptr(out), ptr(err), stream_ptr()), "gtg_embed_dropout_fwd")
        if err is not None and int(err.item()):
            raise _lib.GtgError("embed_dropout: a token id lies outside the embedding table")
        ctx.save_for_backward(ids_c)
        ctx.weight = weight
        ctx.key = (float(p), seed, sid, V, D, B, a is not None)
        return out

    check_ids = False   # reading the flag back is a host sync: for tests and debugging

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dout):
        L = _lib.lib()
        (ids,) = ctx.saved_tensors
        p, seed, sid, V, D, B, has_add = ctx.key
        dout = _f32c(dout)
        R = ids.numel()
        weight = ctx.weight
        need_w, need_add = ctx.needs_input_grad[1], has_add and ctx.needs_input_grad[2]
        dw_ret = None
        target = None
        if need_w:
            g = weight.grad
            if getattr(weight, "grad_inplace", False) and g is not None and g.is_cuda and g.dtype == torch.float32 \
                    and g.is_contiguous() and g.shape == weight.shape:
                target = g                      # accumulated in place; autograd gets no gradient for the weight
            else:
                target = dw_ret = torch.zeros((V, D), dtype=torch.float32, device=dout.device)
        d_add = torch.empty((B, D), dtype=torch.float32, device=dout.device) if need_add else None
        if target is not None or d_add is not None:
            ws = _ws(L.gtg_embed_dropout_bwd_workspace_bytes(R, V, D, B if need_add else 0), dout.device)
            check(L.gtg_embed_dropout_bwd(ptr(dout), ptr(ids), R, V, D, p, seed, sid, ptr(target), ptr(d_add),
                                          B if need_add else 0, ptr(ws), ws.numel(), stream_ptr()), "gtg_embed_dropout_bwd")
        return None, dw_ret, d_add, None


def embed_dropout(ids, weight, p: float = 0.0, add=None):
    """(T, B, D) = dropout_p(weight[ids]) + add[None]; see EmbedDropoutFn."""
    return EmbedDropoutFn.apply(ids, weight, add, float(p))


class DropoutFn(torch.autograd.Function):
    """nn.Dropout(p) in training mode (text_vae.py:64): y = x * keep / (1 - p), the mask regenerated in backward."""

    @staticmethod
    @_on_tensor_device
    def forward(ctx, x, p):
        x = _f32c(x)
        if x.numel() % 4:
            raise _lib.GtgError("dropout: the element count must be a multiple of 4")
        y = torch.empty_like(x)
        seed, sid = _rng_key()
        check(_lib.lib().gtg_dropout(ptr(x), x.numel(), float(p), seed, sid, ptr(y), stream_ptr()), "gtg_dropout")
        ctx.key = (float(p), seed, sid)
        return y

    @staticmethod
    @_on_tensor_device
    def backward(ctx, dy):
        p, seed, sid = ctx.key
        dy = _f32c(dy)
        dx = torch.empty_like(dy)
        check(_lib.lib().gtg_dropout(ptr(dy), dy.numel(), p, seed, sid, ptr(dx), stream_ptr()), "gtg_dropout")
        return dx, None


def dropout(x, p: float, training: bool = True):
    """x when not training or p == 0, else DropoutFn."""
    if not training or p <= 0.0:
        return x
    return DropoutFn.apply(x, float(p))


# ---------------------------------------------------------------------------
# losses and read-outs on rows of vocabulary logits
# ---------------------------------------------------------------------------
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # GTG_DTYPE_*
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}                      # GTG_REDUCE_*


def _need(ok, msg):
    if not ok:
        raise _lib.GtgError(msg)


def _token_rows(what, logits, targets):
    """(x, y, (dtype code, rows, V, row stride)): the logits as memory of equally spaced rows with unit stride along V, and
    the targets as contiguous int64 -- the tensors themselves where their strides allow it, copies otherwise."""
    code = _DTYPES.get(logits.dtype)
    if code is None or not logits.is_cuda:
        _lib.require_cuda(logits, targets)
        raise _lib.GtgError(f"{what}: logits must be float32, float16 or bfloat16, not {logits.dtype}")
    shape = logits.shape
    _need(len(shape) >= 1 and shape[-1] >= 1, f"{what}: logits must be (..., vocab)")
    V = shape[-1]
    R = logits.numel() // V
    x, ld = logits, V
    if not logits.is_contiguous():
        x = logits if logits.dim() == 2 else logits.reshape(-1, V)
        if (x.stride(1) != 1 and V > 1) or (x.stride(0) < V and R > 1):
            x = x.contiguous()
        elif R > 1:
            ld = x.stride(0)
    if targets is not None:
        _lib.require_cuda(targets)
        _need(targets.shape == shape[:-1], f"{what}: targets {tuple(targets.shape)} do not match logits {tuple(shape)}")
        _same_device(what, x, targets)
        if targets.dtype != torch.int64:
            _need(not (targets.is_floating_point() or targets.is_complex() or targets.dtype == torch.bool),
                  f"{what}: targets must be integers")
            targets = targets.long()
        targets = targets.contiguous()
    return x, targets, (code, R, V, ld)


def _same_device(what, x, *others):
    for t in others:
        if t is not None and t.device != x.device:
            raise _lib.GtgError(f"{what}: every tensor must be on the logits' device ({x.device}), not on {t.device}")


def _row_floats(what, name, t, x, shape):
    """A float tensor of the rows' shape as contiguous fp32 on the logits' device."""
    _need(torch.is_tensor(t) and t.is_floating_point(), f"{what}: {name} must be a floating tensor")
    _same_device(what, x, t)
    _need(t.shape == shape, f"{what}: {name} must be {tuple(shape)}, not {tuple(t.shape)}")
    return (t if t.dtype == torch.float32 else t.float()).contiguous()


def _mask_bytes(what, mask, x, shape):
    if mask is None:
        return None
    _same_device(what, x, mask)
    _need(mask.shape == shape, f"{what}: mask must be {tuple(shape)}, not {tuple(mask.shape)}")
    return (mask if mask.dtype == torch.bool else mask != 0).contiguous().view(torch.uint8)


def _grad_like(x, shape, rows):
    """(uninitialised gradient of the logits' shape and type, its row stride): its rows have the alignment of x's rows
    modulo 16 bytes, so that the kernels read and write whole 16-byte vectors; contiguous where x's rows allow that."""
    _, R, V, ld = rows
    size = x.element_size()
    vec = 16 // size
    skew, off = (ld - V) % vec, x.data_ptr() % 16 // size
    if skew == 0 and off == 0:
        return torch.empty(shape, dtype=x.dtype, device=x.device), V
    buf = torch.empty((R * (V + skew) + vec,), dtype=x.dtype, device=x.device)
    return buf[off:off + R * (V + skew)].view(R, V + skew)[:, :V].view(shape), V + skew


def _float_arg(what, name, v):
    _need(isinstance(v, (int, float)), f"{what}: {name} must be a number")
    return float(v)


def _opt(t):
    return None if t is None else t.data_ptr()


@_on_tensor_device
def top_logits(logits, k: int, temperature: float = 1.0):
    """A teacher's answer in short: the k largest logits of every row of (..., V) in descending order -- equal ones by
    ascending index, a NaN above every number -- and the log mass of the rest.

    Returns (values (..., k) of the logits' type, indices (..., k) int32, tail (...) fp32), tail = log sum exp(logits /
    temperature) over the classes that were not selected (-inf where k == V).  1 <= k <= min(V, 256).  No gradient.
    What ``distill_loss`` takes of a teacher."""
    x, _, rows = _token_rows("top_logits", logits.detach() if logits.requires_grad else logits, None)
    _need(isinstance(k, int) and 1 <= k <= min(256, rows[2]), "top_logits: k must be an integer in [1, min(vocab, 256)]")
    lead, dev = logits.shape[:-1], x.device
    values = torch.empty(lead + (k,), dtype=x.dtype, device=dev)
    indices = torch.empty(lead + (k,), dtype=torch.int32, device=dev)
    tail = torch.empty(lead, dtype=torch.float32, device=dev)
    rc = _lib.lib().gtg_top_logits(x.data_ptr(), *rows, k, _float_arg("top_logits", "temperature", temperature), values.data_ptr(),
                                   indices.data_ptr(), tail.data_ptr(), stream_ptr())
    if rc:
        check(rc, "gtg_top_logits")
    return values, indices, tail


def _grad_wanted(logits):
    """Whether a call records a gradient: without one the library is called past autograd (4 us less per call)."""
    return torch.is_grad_enabled() and logits.requires_grad


# The autograd functions below take the logits and one plain tuple with everything else (tensors among it, which get no
# gradient): autograd looks at every argument of a call, and a call on a small batch lasts no longer than that.


@_on_tensor_device
def _token_logprob(logits, targets, padidx, temperature, stats_too):
    x, y, rows = _token_rows("token_logprob", logits, targets)
    temperature = _float_arg("token_logprob", "temperature", temperature)
    logp = torch.empty(targets.shape, dtype=torch.float32, device=x.device)
    entropy = torch.empty_like(logp)
    stats = torch.empty((rows[1], 4), dtype=torch.float32, device=x.device) if stats_too else None
    rc = _lib.lib().gtg_token_logprob_fwd(x.data_ptr(), *rows, y.data_ptr(), int(padidx), temperature, logp.data_ptr(),
                                          entropy.data_ptr(), _opt(stats), stream_ptr())
    if rc:
        check(rc, "gtg_token_logprob_fwd")
    return logp, entropy, (x, y, stats), (int(padidx), temperature, logits.shape, rows)


class TokenLogprobFn(torch.autograd.Function):
    """(log softmax(logits / temperature)[target], entropy of that distribution) per row, zeros where the target is
    padidx; both differentiable.  The backward reads the logits once more and keeps four numbers per row."""

    @staticmethod
    def forward(ctx, logits, args):
        logp, entropy, saved, ctx.key = _token_logprob(logits, *args, True)
        ctx.save_for_backward(*saved)
        ctx.set_materialize_grads(False)
        return logp, entropy

    @staticmethod
    @torch.autograd.function.once_differentiable
    @_on_tensor_device
    def backward(ctx, g_logp, g_entropy):
        if g_logp is None and g_entropy is None:
            return None, None
        x, y, stats = ctx.saved_tensors
        padidx, temperature, shape, rows = ctx.key
        g_logp, g_entropy = _f32c(g_logp), _f32c(g_entropy)
        dx, ldg = _grad_like(x, shape, rows)
        rc = _lib.lib().gtg_token_logprob_bwd(x.data_ptr(), *rows, y.data_ptr(), padidx, temperature, stats.data_ptr(), _opt(g_logp),
                                              _opt(g_entropy), dx.data_ptr(), ldg, stream_ptr())
        if rc:
            check(rc, "gtg_token_logprob_bwd")
        return dx, None


def token_logprob(logits, targets, padidx, temperature: float = 1.0):
    """(logp, entropy), each of targets' shape: log softmax(logits / temperature) at the target and the entropy of that
    distribution; logits (..., V) fp32, fp16 or bf16, targets (...) integers.  Rows whose target is padidx give zero, a
    target outside the vocabulary NaN.  See TokenLogprobFn."""
    if _grad_wanted(logits):
        return TokenLogprobFn.apply(logits, (targets, padidx, temperature))
    return _token_logprob(logits, targets, padidx, temperature, False)[:2]


@_on_tensor_device
def _row_loss_fwd(logits, op, args, reduction, with_grad):
    """The forward of a row loss (`op`: _DistillLoss or _PolicyLoss): (outputs, tensors for the backward, the gradient for an
    upstream gradient of 1 or None, the rest for the backward)."""
    x, y, rows = _token_rows(op.NAME, logits, args[0])
    code = _REDUCTIONS.get(reduction)
    _need(code is not None, f"{op.NAME}: reduction must be one of {sorted(_REDUCTIONS)}")
    saved, scalars = op.check(x, args)
    lead, shape, dev = args[0].shape, logits.shape, x.device
    dx, ldg = _grad_like(x, shape, rows) if code and with_grad else (None, rows[2])
    if code:   # the mean's factor (8 bytes), then a loss per row
        ws = torch.empty((rows[1] + 4,), dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        at = ws.data_ptr()
        norm, row_loss, total = at if code == 2 else None, at + 16, loss.data_ptr()
    else:
        ws, loss, norm, total = None, torch.empty(lead, dtype=torch.float32, device=dev), None, None
        row_loss = loss.data_ptr()
    outputs = (loss,) + op.outputs(lead, dev)
    rc = op.fwd()(x.data_ptr(), *rows, y.data_ptr(), *op.pointers(saved, scalars), code, norm, row_loss, total,
                  *[t.data_ptr() for t in outputs[1:]], None if dx is None else dx.data_ptr(), ldg, stream_ptr())
    if rc:
        check(rc, op.NAME)
    return outputs, (x, y, ws) + saved, dx, (op, scalars, code, ldg, shape, rows)


class RowLossFn(torch.autograd.Function):
    """What the distillation and the policy loss share: a loss per row of logits and its gradient from one sweep.

    With a scalar reduction and ``eager_grad`` the forward writes the logits' gradient for an upstream gradient of 1
    along with the loss -- one read and one write of the logits' size in all -- and the backward hands that out: it
    launches the gradient sweep again on condition that the upstream gradient, known on the device only, is not 1.
    Without ``eager_grad``, and for reduction "none", the gradient is computed in the backward alone (two reads, one
    write).  A second backward through a retained graph computes it anew."""

    @staticmethod
    def forward(ctx, logits, call):
        outputs, saved, ctx.dx, ctx.rest = _row_loss_fwd(logits, *call)
        ctx.save_for_backward(*saved)
        if len(outputs) == 1:
            return outputs[0]
        ctx.mark_non_differentiable(*outputs[1:])
        ctx.set_materialize_grads(False)
        return outputs

    @staticmethod
    @torch.autograd.function.once_differentiable
    @_on_tensor_device
    def backward(ctx, g, *_):
        if g is None:
            return None, None
        x, y, ws, *saved = ctx.saved_tensors
        op, scalars, code, ldg, shape, rows = ctx.rest
        g = _f32c(g)
        dx, ctx.dx = ctx.dx, None          # handed out once: afterwards it is the receiver's
        have = dx is not None
        if not have:
            dx, ldg = _grad_like(x, shape, rows)
        rc = op.bwd()(x.data_ptr(), *rows, y.data_ptr(), *op.pointers(saved, scalars), ws.data_ptr() if code == 2 else None,
                      None if code else g.data_ptr(), g.data_ptr() if code else None, int(have), dx.data_ptr(), ldg, stream_ptr())
        if rc:
            check(rc, op.NAME)
        return dx, None


class _DistillLoss:
    """distill_loss's part of RowLossFn; args: (targets, values, indices, padidx, tail, temperature, ce_weight)."""

    NAME = "distill_loss"
    fwd = staticmethod(lambda: _lib.lib().gtg_distill_loss_fwd)
    bwd = staticmethod(lambda: _lib.lib().gtg_distill_loss_bwd)

    @staticmethod
    def check(x, args):
        what = "distill_loss"
        targets, values, indices, padidx, tail, temperature, ce_weight = args
        lead, shape = targets.shape, values.shape
        _need(values.dtype in _DTYPES and len(shape) == len(lead) + 1 and shape[:-1] == lead and 1 <= shape[-1] <= 256,
              f"{what}: values must be {tuple(lead) + ('k',)}, k in [1, 256], float32, float16 or bfloat16")
        _need(indices.dtype in (torch.int32, torch.int64) and indices.shape == shape,
              f"{what}: indices must be int32 or int64 of values' shape")
        _same_device(what, x, values, indices)
        if indices.dtype == torch.int64:
            # (what does not fit stays out of range, on its side)
            indices = indices.clamp(-1, 2 ** 31 - 1).int()
        if tail is not None:
            tail = _row_floats(what, "tail", tail, x, lead)
        return ((values.contiguous(), indices.contiguous(), tail),
                (int(padidx), _float_arg(what, "temperature", temperature), _float_arg(what, "ce_weight", ce_weight)))

    @staticmethod
    def outputs(lead, dev):
        return ()

    @staticmethod
    def pointers(saved, scalars):
        values, indices, tail = saved
        padidx, temperature, ce_weight = scalars
        return (padidx, values.data_ptr(), _DTYPES[values.dtype], indices.data_ptr(), values.shape[-1],
                None if tail is None else tail.data_ptr(), temperature, ce_weight)


def distill_loss(logits, values, indices, targets, padidx, tail=None, temperature: float = 1.0, ce_weight: float = 0.0,
                 reduction: str = "mean", eager_grad: bool = True):
    """Distillation of a teacher's top logits: per row

        (1 - ce_weight) temperature^2 KL(q || p) + ce_weight (-log softmax(logits)[target])

    q is the teacher's distribution over the k classes it lists -- values (..., k), indices (..., k), as ``top_logits``
    gives them -- and, with ``tail`` (...), over "any other class", whose log mass at this temperature tail is; p is the
    student's softmax(logits / temperature) over the same classes and the rest as one.  Without a tail the list is taken
    for the teacher's whole distribution.  A negative index takes no part (a shorter list), one past the vocabulary gives
    NaN; rows whose target is padidx take no part.

    reduction: "mean" over the rows that count (0 if there are none), "sum", or "none" (a loss per row).  Differentiable
    in the logits alone.  ``eager_grad=False`` for a scalar loss that will be scaled before its backward -- by a gradient
    scaler, a number of accumulation steps -- : the gradient is then computed in the backward only, see RowLossFn.
    The divergence is a difference of fp32 sums' logarithms: off by some 2^-20, times temperature^2 in the loss."""
    args = (targets, values, indices, padidx, tail, temperature, ce_weight)
    if _grad_wanted(logits):
        return RowLossFn.apply(logits, (_DistillLoss, args, reduction, eager_grad))
    return _row_loss_fwd(logits, _DistillLoss, args, reduction, False)[0][0]


class _PolicyLoss:
    """policy_loss's part of RowLossFn; args: (targets, padidx, old_logp, advantages, ref_logp, mask, clip_low, clip_high,
    kl_coef, entropy_coef, temperature)."""

    NAME = "policy_loss"
    fwd = staticmethod(lambda: _lib.lib().gtg_policy_loss_fwd)
    bwd = staticmethod(lambda: _lib.lib().gtg_policy_loss_bwd)
    NUMBERS = ("clip_low", "clip_high", "kl_coef", "entropy_coef", "temperature")

    @staticmethod
    def check(x, args):
        what = "policy_loss"
        targets, padidx, old_logp, advantages, ref_logp, mask, *numbers = args
        lead = targets.shape
        old = _row_floats(what, "old_logp", old_logp, x, lead)
        _need(torch.is_tensor(advantages), f"{what}: advantages must be a floating tensor")
        per_column = len(lead) == 2 and advantages.shape == lead[1:]
        adv = _row_floats(what, "advantages", advantages, x, lead[1:] if per_column else lead)
        ref = None if ref_logp is None else _row_floats(what, "ref_logp", ref_logp, x, lead)
        numbers = tuple([_float_arg(what, n, v) for n, v in zip(_PolicyLoss.NUMBERS, numbers)])
        _need(numbers[2] == 0.0 or ref is not None, f"{what}: kl_coef needs ref_logp")
        return (old, adv, ref, _mask_bytes(what, mask, x, lead)), (int(padidx), numbers)

    @staticmethod
    def outputs(lead, dev):
        logp = torch.empty(lead, dtype=torch.float32, device=dev)
        return logp, torch.empty_like(logp)

    @staticmethod
    def pointers(saved, scalars):
        old, adv, ref, mask = saved
        padidx, numbers = scalars
        return (padidx, None if mask is None else mask.data_ptr(), old.data_ptr(), adv.data_ptr(), adv.numel(),
                None if ref is None else ref.data_ptr()) + numbers


def policy_loss(logits, targets, padidx, old_logp, advantages, ref_logp=None, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, entropy_coef: float = 0.0, temperature: float = 1.0, mask=None, reduction: str = "mean",
                eager_grad: bool = True):
    """Clipped policy loss of sampled tokens.  Per row, with logp = log softmax(logits / temperature)[target] and rho =
    exp(logp - old_logp):

        -min(rho A, clip(rho, 1 - clip_low, 1 + clip_high) A) - entropy_coef entropy
        + kl_coef (exp(ref_logp - logp) - (ref_logp - logp) - 1)

    targets, old_logp, ref_logp, mask (...); advantages (...), or (B) for time-major (T, B) targets.  Rows whose target is
    padidx or whose mask is false (a prompt's tokens) take no part.  Returns (loss, logp, entropy), the last two of
    targets' shape and without gradient; reduction and eager_grad as in distill_loss.  Differentiable in the logits
    alone."""
    args = (targets, padidx, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef, entropy_coef, temperature)
    if _grad_wanted(logits):
        return RowLossFn.apply(logits, (_PolicyLoss, args, reduction, eager_grad))
    return _row_loss_fwd(logits, _PolicyLoss, args, reduction, False)[0]


class PreferenceLossFn(torch.autograd.Function):
    """Preference loss over pairs of sequences; see preference_loss.  The weight of every row's gradient depends on both
    whole sequences, so the backward reads the logits once more."""

    @staticmethod
    @_on_tensor_device
    def _forward(logits, targets, padidx, ref_logp, beta, label_smoothing, mask, batch_first, reduction):
        what = "preference_loss"
        x, y, rows = _token_rows(what, logits, targets)
        _need(targets.dim() == 2, f"{what}: targets must be (T, 2 P), or (2 P, T) with batch_first")
        reduce_code = _REDUCTIONS.get(reduction)
        _need(reduce_code is not None, f"{what}: reduction must be one of {sorted(_REDUCTIONS)}")
        S, T = targets.shape if batch_first else targets.shape[::-1]
        _need(S % 2 == 0, f"{what}: an even number of sequences is needed, the chosen ones first, then the rejected ones")
        ref = _row_floats(what, "ref_logp", ref_logp, x, (S,))
        m = _mask_bytes(what, mask, x, targets.shape)
        beta, label_smoothing = _float_arg(what, "beta", beta), _float_arg(what, "label_smoothing", label_smoothing)
        L, dev, P = _lib.lib(), x.device, S // 2
        code, R, V, ld = rows
        # for the backward: four numbers per row and one per sequence; for this call alone: its workspace
        state = torch.empty((4 * R + S,), dtype=torch.float32, device=dev)
        nbytes = L.gtg_preference_workspace_bytes(T, P)
        ws = torch.empty((nbytes + 8,), dtype=torch.uint8, device=dev)
        seq_logp = torch.empty((S,), dtype=torch.float32, device=dev)
        pair_loss = torch.empty((P,), dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev) if reduce_code else None
        head = (code, T, P, V, ld, int(bool(batch_first)))
        rc = L.gtg_preference_fwd(x.data_ptr(), *head, y.data_ptr(), int(padidx), _opt(m), ref.data_ptr(), beta, label_smoothing,
                                  reduce_code, state.data_ptr(), state.data_ptr() + 16 * R, seq_logp.data_ptr(),
                                  pair_loss.data_ptr(), _opt(loss), ws.data_ptr(), nbytes, stream_ptr())
        if rc:
            check(rc, "gtg_preference_fwd")
        return pair_loss if loss is None else loss, seq_logp, (x, y, m, state), (head, int(padidx), loss is not None, logits.shape, rows)

    @staticmethod
    def forward(ctx, logits, args):
        loss, seq_logp, saved, ctx.call = PreferenceLossFn._forward(logits, *args)
        ctx.save_for_backward(*saved)
        ctx.mark_non_differentiable(seq_logp)
        ctx.set_materialize_grads(False)
        return loss, seq_logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    @_on_tensor_device
    def backward(ctx, g, _gseq):
        if g is None:
            return None, None
        x, y, m, state = ctx.saved_tensors
        head, padidx, scalar, shape, rows = ctx.call
        g = _f32c(g)
        dx, ldg = _grad_like(x, shape, rows)
        rc = _lib.lib().gtg_preference_bwd(x.data_ptr(), *head, y.data_ptr(), padidx, _opt(m), state.data_ptr(),
                                           state.data_ptr() + 16 * rows[1], g.data_ptr() if scalar else None,
                                           None if scalar else g.data_ptr(), dx.data_ptr(), ldg, stream_ptr())
        if rc:
            check(rc, "gtg_preference_bwd")
        return dx, None


def preference_loss(logits, targets, padidx, ref_logp, beta: float = 0.1, label_smoothing: float = 0.0, mask=None,
                    batch_first: bool = False, reduction: str = "mean"):
    """Loss of preferred over rejected sequences.  logits (T, 2 P, V) and targets (T, 2 P), time-major as the decoder
    gives them ((2 P, T, V) and (2 P, T) with batch_first): sequence b < P was chosen over sequence P + b.  With seq_logp the
    sums of the tokens' log-probabilities over each sequence (targets equal to padidx, and tokens whose mask is false,
    left out), ref_logp (2 P) the same sums under the reference model, and margin = beta ((seq_logp - ref_logp)[chosen] -
    (seq_logp - ref_logp)[rejected]):

        -(1 - label_smoothing) log sigma(margin) - label_smoothing log sigma(-margin)

    Returns (loss, seq_logp (2 P), without gradient); reduction over the pairs: "mean", "sum" or "none".  Differentiable
    in the logits alone."""
    args = (targets, padidx, ref_logp, beta, label_smoothing, mask, batch_first, reduction)
    return PreferenceLossFn.apply(logits, args) if _grad_wanted(logits) else PreferenceLossFn._forward(logits, *args)[:2]
