"""torch view of the device operators that belong to no index (include/jvgpu.h, "training and 8-bit scoring of vectors"):

* ``encode_blocks`` / ``decode_blocks`` / ``score_blocks`` — rows of 8-bit floats (e4m3) with a power-of-two scale for each block of 128
  components, and the matrix product of a batch of queries with such rows;
* ``softmax_loss`` / ``softmax_loss_grad`` — softmax cross entropy of queries over all rows of a matrix, without keeping the logits, and
  its gradient: what an embedding model or a query adapter is trained with against a corpus.

Plumbing only: argument checks, output tensors and workspaces from torch's allocator, the calls of the C ABI on torch's current
stream of the tensors' device (which need not be the current device).  Nothing here waits for the GPU or keeps anything between calls, so
every function can be captured into a graph; there is no CPU fallback.  Vectors are float32 or bfloat16 matrices whose rows are
contiguous; the rows may lie any distance apart.  Not differentiable by autograd: the gradient is a call of its own, and a loss of tensors that
autograd records is refused (detach them, or call under ``torch.no_grad()``).
"""
from __future__ import annotations

import functools

import torch

from . import binding

BLOCK = 128
_DTYPES = {torch.float32: binding.DTYPE_F32, torch.bfloat16: binding.DTYPE_BF16}
_LEGACY_STREAM = 1   # hipStreamLegacy: the default stream's handle (0) would make the call wait for its work


def _stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index) or _LEGACY_STREAM   # (what current_stream(device).cuda_stream is, without its objects)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(dtype: int, nq: int, n: int, d: int, flags: int, offset: int, odd: bool) -> int:
    # the shape decides, and whether the vectors can be taken as they lie: `offset`: their address to 4 bytes, `odd`: their stride
    params = binding.softmax_params(0, dtype, nq, n, d, 1.0, d_vectors=4 + offset, vector_stride=int(odd))
    return binding.softmax_workspace(params, flags | binding.SOFTMAX_AS_THEY_LIE)


def _matrix(x: torch.Tensor, what: str, name: str):
    """(dtype, rows, components, row stride) of a matrix of vectors."""
    if x.dim() != 2 or not x.is_cuda:
        raise ValueError(f"{what}: {name}: a 2-D tensor on a GPU is wanted, got shape {tuple(x.shape)} on {x.device}")
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"{what}: {name}: float32 or bfloat16 is wanted, got {x.dtype}")
    n, d = x.shape
    apart, step = x.stride()
    if step != 1 and d > 1 and n > 0:
        raise ValueError(f"{what}: {name}: the components of a row have to be contiguous, got strides {x.stride()}")
    return dtype, n, d, apart if n > 1 else d


def _like(x: torch.Tensor, device, shape, dtype, what: str, name: str):
    if x.dtype is not dtype or x.shape != shape or x.device != device or not x.is_contiguous():
        raise ValueError(f"{what}: {name}: a contiguous {dtype} tensor of shape {tuple(shape)} on {device} is wanted, got {x.dtype} {tuple(x.shape)} on {x.device}")


def _codes(codes: torch.Tensor, scales: torch.Tensor, d: int, what: str) -> int:
    blocks = -(-d // BLOCK)
    if codes.dim() != 2 or not codes.is_cuda:
        raise ValueError(f"{what}: 2-D codes on a GPU are wanted")
    n, device = codes.shape[0], codes.device
    _like(codes, device, (n, blocks * BLOCK), torch.uint8, what, "codes")
    _like(scales, device, (n, blocks), torch.uint8, what, "scales")
    return n


def encode_blocks(vectors: torch.Tensor):
    """(codes [n][blocks * 128] uint8, scales [n][blocks] uint8) of [n][d] vectors; see jv_encode_blocks_device."""
    dtype, n, d, stride = _matrix(vectors, "encode_blocks", "vectors")
    dev, blocks = vectors.device, -(-d // BLOCK)
    codes = vectors.new_empty((n, blocks * BLOCK), dtype=torch.uint8)
    scales = vectors.new_empty((n, blocks), dtype=torch.uint8)
    binding.encode_blocks_device(dev.index, vectors.data_ptr(), dtype, stride, n, d, codes.data_ptr(), scales.data_ptr(), _stream(dev))
    return codes, scales


def decode_blocks(codes: torch.Tensor, scales: torch.Tensor, d: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[n][d] values that the codes stand for; see jv_decode_blocks_device."""
    n = _codes(codes, scales, d, "decode_blocks")
    if dtype not in _DTYPES:
        raise ValueError(f"decode_blocks: float32 or bfloat16 is wanted, got {dtype}")
    out = codes.new_empty((n, d), dtype=dtype)
    binding.decode_blocks_device(codes.device.index, codes.data_ptr(), scales.data_ptr(), n, d, _DTYPES[dtype], out.data_ptr(), d, _stream(codes.device))
    return out


def score_blocks(query_codes: torch.Tensor, query_scales: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, d: int,
                 dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[nq][n] dot products of encoded queries with encoded rows; see jv_score_blocks_device."""
    nq, n = _codes(query_codes, query_scales, d, "score_blocks: queries"), _codes(codes, scales, d, "score_blocks: rows")
    if query_codes.device != codes.device or dtype not in _DTYPES:
        raise ValueError("score_blocks: queries and rows on one device and float32 or bfloat16 scores are wanted")
    out = codes.new_empty((nq, n), dtype=dtype)
    binding.score_blocks_device(codes.device.index, query_codes.data_ptr(), query_scales.data_ptr(), nq, codes.data_ptr(), scales.data_ptr(), n, d,
                                _DTYPES[dtype], out.data_ptr(), n, _stream(codes.device))
    return out


def _softmax(queries, vectors, targets, scale, what, flags):
    """(params with a workspace, the workspace, the device) of a softmax call."""
    dtype, nq, d, q_stride = _matrix(queries, what, "queries")
    v_dtype, n, v_d, v_stride = _matrix(vectors, what, "vectors")
    device = queries.device
    if v_dtype != dtype or v_d != d or vectors.device != device:
        raise ValueError(f"{what}: queries {queries.dtype} {tuple(queries.shape)} on {queries.device} and vectors {vectors.dtype} "
                         f"{tuple(vectors.shape)} on {vectors.device} do not match")
    if targets is not None:
        _like(targets, device, (nq,), torch.int32, what, "targets")
    params = binding.softmax_params(device.index, dtype, nq, n, d, scale, queries.data_ptr(), q_stride, vectors.data_ptr(), v_stride,
                                    0 if targets is None else targets.data_ptr())
    need = _workspace_bytes(dtype, nq, n, d, flags, vectors.data_ptr() % 4, v_stride % 2 == 1)
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    params.workspace_bytes, params.workspace = need, workspace.data_ptr()
    return params, workspace, device


def softmax_loss(queries: torch.Tensor, vectors: torch.Tensor, targets, scale: float):
    """(loss [nq], lse [nq]), float32: loss_i = lse_i - scale q_i . v_targets[i], lse_i = log sum_j exp(scale q_i . v_j).  ``targets``: int32, a value
    outside [0, n) (or None in place of the tensor) = no target, loss 0; see jv_softmax_loss_device."""
    if torch.is_grad_enabled() and (queries.requires_grad or vectors.requires_grad):
        raise ValueError("softmax_loss: autograd does not see this loss: detach the queries and vectors, or call it under torch.no_grad(), and take the gradient "
                         "from softmax_loss_grad")
    params, workspace, device = _softmax(queries, vectors, targets, scale, "softmax_loss", binding.SOFTMAX_LOSS)
    nq = queries.shape[0]
    loss = torch.empty(nq, dtype=torch.float32, device=device)
    lse = torch.empty(nq, dtype=torch.float32, device=device)
    binding.softmax_loss_device(params, loss.data_ptr(), lse.data_ptr(), _stream(device))
    return loss, lse


def softmax_loss_grad(queries: torch.Tensor, vectors: torch.Tensor, targets, scale: float, lse: torch.Tensor, loss_grad=None, queries_grad: bool = True,
                      vectors_grad: bool = True, loss=None):
    """Gradients of sum_i loss_grad[i] * loss[i] (``loss_grad`` None = 1 each) by the queries and by the vectors, in their dtype; None in the place
    of one that is not asked for.  ``lse`` and ``loss`` as ``softmax_loss`` returned them; without ``loss`` the gradient of a pair that is nearly
    learnt keeps only the digits that a float32 lse leaves (two at a loss of 1e-4); see jv_softmax_grad_device."""
    if not queries_grad and not vectors_grad:
        return None, None
    flags = (binding.SOFTMAX_QUERY_GRAD if queries_grad else 0) | (binding.SOFTMAX_VECTOR_GRAD if vectors_grad else 0)
    params, workspace, device = _softmax(queries, vectors, targets, scale, "softmax_loss_grad", flags)
    nq, d = queries.shape
    _like(lse, device, (nq,), torch.float32, "softmax_loss_grad", "lse")
    if loss is not None:
        _like(loss, device, (nq,), torch.float32, "softmax_loss_grad", "loss")
    if loss_grad is not None:
        _like(loss_grad, device, (nq,), torch.float32, "softmax_loss_grad", "loss_grad")
    dq = queries.new_empty((nq, d)) if queries_grad else None
    dv = vectors.new_empty(vectors.shape) if vectors_grad else None
    # (an empty tensor has no address: its gradient has nothing to write either)
    if (dq is None or dq.numel() == 0) and (dv is None or dv.numel() == 0):
        return dq, dv
    binding.softmax_grad_device(params, lse.data_ptr(), 0 if loss_grad is None else loss_grad.data_ptr(), 0 if dq is None else dq.data_ptr(),
                                d, 0 if dv is None else dv.data_ptr(), d, _stream(device), 0 if loss is None else loss.data_ptr())
    return dq, dv
