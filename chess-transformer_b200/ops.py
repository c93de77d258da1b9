"""The reference's torch custom ops, one by one, on libfry_b200.so (torch.library ops in the `fry` namespace).

Each keeps the reference op's name, argument meaning, output shapes and dtypes (model/int8_blocks.py:132-251,
model/fused_blocks.py:104-177,308-318,397-411,495-512,743-779) and runs on the caller's current CUDA stream, so the ops
can be recorded in CUDA graphs and seen through by torch.compile (each has a fake implementation). CPU tensors are
refused with FryError: there is no CPU path.
"""
import ctypes
import functools

import torch

from .library import FryError, FryHeads, library

HADAMARD_BLOCK = 32


def _stream(tensor: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(tensor.device).cuda_stream)


def _ptr(tensor: torch.Tensor | None) -> ctypes.c_void_p | None:
    return None if tensor is None else ctypes.c_void_p(tensor.data_ptr())


def _cuda(name: str, *tensors: torch.Tensor | None) -> None:
    for tensor in tensors:
        if tensor is not None and not tensor.is_cuda:
            raise FryError(f"{name} runs on the GPU only; got a tensor on {tensor.device}")


def _dtype(name: str, tensor: torch.Tensor | None, dtype: torch.dtype, what: str) -> None:
    if tensor is not None and tensor.dtype != dtype:
        raise FryError(f"{name}: {what} must be {dtype}, got {tensor.dtype}")


@torch.library.custom_op("fry::int8_linear", mutates_args=())
def int8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None,
                residual: torch.Tensor | None, gated: bool, matmul: str, original: torch.Tensor | None = None,
                residual_scale: torch.Tensor | None = None, input_scale: torch.Tensor | None = None) -> torch.Tensor:
    """`chess::int8_linear` (model/int8_blocks.py:132-139). `matmul` names the reference's tile table; one kernel serves all."""
    _cuda("int8_linear", x, x_scale, weight, weight_scale, bias, residual, original)
    _dtype("int8_linear", x, torch.int8, "x")
    _dtype("int8_linear", weight, torch.int8, "weight")
    rows, K = weight.shape
    N = rows // 2 if gated else rows
    x = x.contiguous()
    M = x.numel() // K
    out = torch.empty(*x.shape[:-1], N, device=x.device, dtype=torch.float16)
    residual = residual.contiguous() if residual is not None else None
    original = original.contiguous() if original is not None else None
    x_scale, weight, weight_scale = x_scale.contiguous().float(), weight.contiguous(), weight_scale.contiguous().float()
    bias = bias.half().contiguous() if bias is not None else None
    library().fry_int8_linear(_ptr(x), _ptr(x_scale), _ptr(weight), _ptr(weight_scale), _ptr(bias), _ptr(residual), _ptr(original),
                              _ptr(residual_scale), _ptr(input_scale), _ptr(out), M, N, K, int(gated), _stream(x))
    return out


@int8_linear.register_fake
def _(x, x_scale, weight, weight_scale, bias, residual, gated, matmul, original=None, residual_scale=None, input_scale=None):
    return x.new_empty(*x.shape[:-1], weight.shape[0] // 2 if gated else weight.shape[0], dtype=torch.float16)


@torch.library.custom_op("fry::int8_linear_normed", mutates_args=())
def int8_linear_normed(x: torch.Tensor, gain: torch.Tensor, eps: float, weight: torch.Tensor, weight_scale: torch.Tensor,
                       bias: torch.Tensor | None, gated: bool) -> torch.Tensor:
    """`chess::norm_quant` then `chess::int8_linear` (model/int8_blocks.py:191-193, :132-139) as one kernel, the pair
    `Int8Block.forward` runs for ln1 -> projection and ln2 -> gate_up (model/int8_blocks.py:274-288); the same bits as
    `int8_linear(*norm_quant(x, gain, eps), ...)`. x fp16 [..., 768]."""
    _cuda("int8_linear_normed", x, gain, weight, weight_scale, bias)
    _dtype("int8_linear_normed", x, torch.float16, "x")
    _dtype("int8_linear_normed", weight, torch.int8, "weight")
    rows, K = weight.shape
    N = rows // 2 if gated else rows
    x = x.contiguous()
    M = x.numel() // K
    out = torch.empty(*x.shape[:-1], N, device=x.device, dtype=torch.float16)
    bias = bias.half().contiguous() if bias is not None else None
    library().fry_int8_linear_normed(_ptr(x), _ptr(gain.half().contiguous()), eps, _ptr(weight.contiguous()),
                                     _ptr(weight_scale.contiguous().float()), _ptr(bias), _ptr(out), M, N, K, int(gated), _stream(x))
    return out


@int8_linear_normed.register_fake
def _(x, gain, eps, weight, weight_scale, bias, gated):
    return x.new_empty(*x.shape[:-1], weight.shape[0] // 2 if gated else weight.shape[0], dtype=torch.float16)


@torch.library.custom_op("fry::int8_matmul_i32", mutates_args=())
def int8_matmul_i32(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """The int32 sums x . weight^T of the int8 tensor-core kernel (what int8_linear's epilogue starts from)."""
    _cuda("int8_matmul_i32", x, weight)
    x, weight = x.contiguous(), weight.contiguous()
    N, K = weight.shape
    M = x.numel() // K
    out = torch.empty(*x.shape[:-1], N, device=x.device, dtype=torch.int32)
    library().fry_int8_matmul_i32(_ptr(x), _ptr(weight), _ptr(out), M, N, K, _stream(x))
    return out


@int8_matmul_i32.register_fake
def _(x, weight):
    return x.new_empty(*x.shape[:-1], weight.shape[0], dtype=torch.int32)


@torch.library.custom_op("fry::int8_matmul_scaled_bf16", mutates_args=())
def int8_matmul_scaled_bf16(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor) -> torch.Tensor:
    """The benchmark's isolated int8 GEMM: bf16((acc * x_scale[m]) * weight_scale[n]), acc = x . weight^T in int32, on the
    int8 tensor-core kernel. x int8 [..., K], weight int8 [N, K], scales fp32."""
    _cuda("int8_matmul_scaled_bf16", x, x_scale, weight, weight_scale)
    _dtype("int8_matmul_scaled_bf16", x, torch.int8, "x")
    _dtype("int8_matmul_scaled_bf16", weight, torch.int8, "weight")
    x, weight = x.contiguous(), weight.contiguous()
    N, K = weight.shape
    M = x.numel() // K
    out = torch.empty(*x.shape[:-1], N, device=x.device, dtype=torch.bfloat16)
    library().fry_int8_matmul_scaled_bf16(_ptr(x), _ptr(x_scale.contiguous().float()), _ptr(weight), _ptr(weight_scale.contiguous().float()),
                                          _ptr(out), M, N, K, _stream(x))
    return out


@int8_matmul_scaled_bf16.register_fake
def _(x, x_scale, weight, weight_scale):
    return x.new_empty(*x.shape[:-1], weight.shape[0], dtype=torch.bfloat16)


@torch.library.custom_op("fry::attention_bf16", mutates_args=())
def attention_bf16(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, heads: int) -> torch.Tensor:
    """The benchmark's isolated attention: softmax(q k^T / 8) v per sequence and head, q, k, v bf16 [B, 64, heads * 64]."""
    _cuda("attention_bf16", q, k, v)
    for name, tensor in (("q", q), ("k", k), ("v", v)):
        _dtype("attention_bf16", tensor, torch.bfloat16, name)
    if q.dim() != 3 or q.shape != k.shape or q.shape != v.shape or q.shape[-1] % heads != 0:
        raise FryError(f"attention_bf16 takes q, k and v of one shape [B, seq, heads * head_dim], got {tuple(q.shape)}")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    B, seq, width = q.shape
    out = torch.empty_like(q)
    library().fry_attention_bf16(_ptr(q), _ptr(k), _ptr(v), _ptr(out), B, heads, seq, width // heads, _stream(q))
    return out


@attention_bf16.register_fake
def _(q, k, v, heads):
    return torch.empty_like(q)


# The packed operators below check a call in one expression and go on; where it does not hold, a second function finds out
# what to say: a small call is bound by host code, of which torch's dispatcher is the larger part.

def _call(function, index: int, *arguments) -> None:
    """A library call on device `index` and its current stream, whatever device is current."""
    if index == torch.cuda.current_device():
        function(*arguments, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            function(*arguments, torch._C._cuda_getCurrentRawStream(index))


def _index32(name: str, tensor: torch.Tensor, what: str, count: int, device: torch.device) -> None:
    if tensor.dtype != torch.int32 or tensor.dim() != 1 or tensor.shape[0] != count or tensor.device != device:
        raise FryError(f"{name}: {what} must be int32 [{count}] on {device}, got {tensor.dtype} {tuple(tensor.shape)} on {tensor.device}")


def _readable(tensor: torch.Tensor) -> tuple[torch.Tensor, list[int]]:
    """A 16-bit tensor as the attention kernels read it, its last axis dense and its other strides and its start on 16
    bytes (a copy if they are not), and those strides. An axis of one has no stride to keep."""
    *strides, unit = tensor.stride()
    if unit == 1 and not tensor.data_ptr() % 16 and all(s and not s % 8 for s in strides):
        return tensor, strides
    strides = [s if n > 1 else 8 for s, n in zip(strides, tensor.shape)]
    if (unit != 1 and tensor.shape[-1] > 1) or any(s % 8 or not s for s in strides) or tensor.data_ptr() % 16:
        tensor = tensor.clone(memory_format=torch.contiguous_format)
        strides = [s if n > 1 else 8 for s, n in zip(tensor.stride()[:-1], tensor.shape)]
    return tensor, strides


_HALVES = (torch.float16, torch.bfloat16)


def _refuse_attention(name: str, q, k, v, shaped: bool, indexes: dict, layout: str) -> None:
    """Says what is wrong with a call of the attention ops."""
    _cuda(name, q, k, v)
    if q.dtype not in _HALVES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise FryError(f"{name}: q, k and v must be of one type, fp16 or bf16, got {q.dtype}, {k.dtype} and {v.dtype}")
    if k.device != q.device or v.device != q.device:
        raise FryError(f"{name}: q, k and v must be on one device, got {q.device}, {k.device} and {v.device}")
    if shaped:
        for what, (tensor, count) in indexes.items():
            _index32(name, tensor, what, count, q.device)
    raise FryError(f"{name} takes {layout}, heads a multiple of kv_heads, got {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(function: str, *shape: int) -> int:
    return getattr(library(), function)(*shape)


@torch.library.custom_op("fry::packed_attention", mutates_args=())
def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_offsets: torch.Tensor, k_offsets: torch.Tensor, causal: bool = True,
                     scale: float | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v over sequences packed one behind the other (the op fry::packed_attention): q [rows, heads,
    width], k and v [key rows, kv_heads, width], fp16 or bf16, query head h on key/value head h // (heads // kv_heads);
    sequence s has the rows q_offsets[s] to q_offsets[s + 1] and the keys k_offsets[s] to k_offsets[s + 1] (int32, on the
    device). Causal, its queries are its last tokens: query i of nq sees keys j <= i + nk - nq. Rows that see no key, and
    rows of no sequence, are 0. width a multiple of 8 up to 128; scale defaults to 1 / sqrt(width). No backward pass.
    Strided views (of a projection's rows, say) are read in place where their last axis is dense and their other strides
    are multiples of 8 other than 0; others are copied first."""
    q_shape, k_shape, dtype, index = q.shape, k.shape, q.dtype, q.get_device()
    shaped = (len(q_shape) == 3 and len(k_shape) == 3 and v.shape == k_shape and q_shape[2] == k_shape[2] and k_shape[1] > 0
              and q_shape[1] % k_shape[1] == 0)
    if not (shaped and dtype in _HALVES and k.dtype is dtype and v.dtype is dtype and index >= 0
            and k.get_device() == v.get_device() == q_offsets.get_device() == k_offsets.get_device() == index
            and q_offsets.dtype is k_offsets.dtype is torch.int32 and q_offsets.dim() == 1 and q_offsets.shape == k_offsets.shape != (0,)):
        count = max(q_offsets.numel(), 1)
        _refuse_attention("packed_attention", q, k, v, shaped, {"q_offsets": (q_offsets, count), "k_offsets": (k_offsets, count)},
                          "q [rows, heads, width] and k and v [key rows, kv_heads, width]")
    (q, (q_row, q_head)), (k, (k_row, k_head)), (v, (v_row, v_head)) = _readable(q), _readable(k), _readable(v)
    rows, heads, width = q_shape
    key_rows, kv_heads, _ = k_shape
    q_offsets, k_offsets = q_offsets.contiguous(), k_offsets.contiguous()
    sequences = q_offsets.shape[0] - 1
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q_shape)
    size = _workspace_bytes("fry_packed_attention_workspace_bytes", rows, key_rows, sequences, heads, kv_heads, width)
    workspace = torch.empty(size, device=q.device, dtype=torch.uint8) if size else None
    _call(library().fry_packed_attention, index, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), q_offsets.data_ptr(),
          k_offsets.data_ptr(), rows, key_rows, sequences, heads, kv_heads, width, q_row, q_head, k_row, k_head, v_row, v_head,
          (width or 1) ** -0.5 if scale is None else scale, causal, dtype is torch.bfloat16, workspace.data_ptr() if size else None, size)
    return out


@packed_attention.register_fake
def _(q, k, v, q_offsets, k_offsets, causal=True, scale=None):
    return q.new_empty(q.shape)


@torch.library.custom_op("fry::cached_attention", mutates_args=())
def cached_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, scale: float | None = None) -> torch.Tensor:
    """packed_attention for one query token a sequence over a cache (the op fry::cached_attention): q [sequences, heads,
    width], k and v [sequences, capacity, kv_heads, width] by any strides, of which sequence s has its first lengths[s] keys
    (int32, on the device). What lies behind a length is not read; a length of 0 answers 0."""
    q_shape, k_shape, dtype, index = q.shape, k.shape, q.dtype, q.get_device()
    shaped = (len(q_shape) == 3 and len(k_shape) == 4 and v.shape == k_shape and k_shape[0] == q_shape[0] and q_shape[2] == k_shape[3]
              and k_shape[2] > 0 and q_shape[1] % k_shape[2] == 0)
    if not (shaped and dtype in _HALVES and k.dtype is dtype and v.dtype is dtype and index >= 0
            and k.get_device() == v.get_device() == lengths.get_device() == index and lengths.dtype is torch.int32 and lengths.shape == q_shape[:1]):
        _refuse_attention("cached_attention", q, k, v, shaped, {"lengths": (lengths, q_shape[0])},
                          "q [sequences, heads, width] and k and v [sequences, capacity, kv_heads, width]")
    (q, (q_row, q_head)), (k, (k_sequence, k_row, k_head)), (v, (v_sequence, v_row, v_head)) = _readable(q), _readable(k), _readable(v)
    sequences, heads, width = q_shape
    _, capacity, kv_heads, _ = k_shape
    lengths = lengths.contiguous()
    out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(q_shape)
    size = _workspace_bytes("fry_cached_attention_workspace_bytes", sequences, capacity, heads, kv_heads, width)
    workspace = torch.empty(size, device=q.device, dtype=torch.uint8) if size else None
    _call(library().fry_cached_attention, index, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lengths.data_ptr(), sequences,
          capacity, heads, kv_heads, width, q_row, q_head, k_sequence, k_row, k_head, v_sequence, v_row, v_head,
          (width or 1) ** -0.5 if scale is None else scale, dtype is torch.bfloat16, workspace.data_ptr() if size else None, size)
    return out


@cached_attention.register_fake
def _(q, k, v, lengths, scale=None):
    return q.new_empty(q.shape)


def _aligned(tensor: torch.Tensor) -> torch.Tensor:
    """Dense rows that start on 16 bytes (a copy if they do not)."""
    tensor = tensor.contiguous()
    return tensor if tensor.data_ptr() % 16 == 0 else tensor.clone()


def _refuse_adapters(name: str, x, weight, bias, residual, down, up, offsets, ids, dtype) -> None:
    """Says what is wrong with a call of the linears with adapters."""
    _cuda(name, x)
    for tensor in (weight, bias, residual, down, up, offsets, ids):
        if tensor is not None and tensor.device != x.device:
            raise FryError(f"{name}: x is on {x.device}, another operand on {tensor.device}")
    _dtype(name, x, dtype, "x")
    _dtype(name, weight, dtype, "weight")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise FryError(f"{name} takes x [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    if down.dim() != 3 or up.dim() != 3 or down.shape[2] != K or up.shape != (down.shape[0], N, down.shape[1]):
        raise FryError(f"{name} takes down [adapters, rank, {K}] and up [adapters, {N}, rank], got {tuple(down.shape)} and {tuple(up.shape)}")
    for tensor, what in ((bias, "bias"), (residual, "residual"), (down, "down"), (up, "up")):
        _dtype(name, tensor, torch.float16, what)
    if bias is not None and tuple(bias.shape) != (N,):
        raise FryError(f"{name}: bias must be [{N}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != (*x.shape[:-1], N):
        raise FryError(f"{name}: residual must be {(*x.shape[:-1], N)}, got {tuple(residual.shape)}")
    requests = ids.shape[0] if ids.dim() == 1 else -1
    _index32(name, ids, "ids", requests, x.device)
    _index32(name, offsets, "offsets", requests + 1, x.device)
    raise FryError(f"{name}: cannot take this call")


def _adapter_operands(name: str, x, weight, bias, residual, down, up, offsets, ids, dtype) -> tuple[int, tuple[int, ...], tuple[torch.Tensor | None, ...]]:
    """(device, (M, N, K, requests, adapters, rank), the operands dense and aligned) of a linear with adapters, or FryError."""
    x_shape, w_shape, down_shape, index, half = x.shape, weight.shape, down.shape, x.get_device(), torch.float16
    if not (index >= 0 and x.dtype is weight.dtype is dtype and down.dtype is up.dtype is half and offsets.dtype is ids.dtype is torch.int32
            and len(w_shape) == 2 and len(x_shape) > 0 and x_shape[-1] == w_shape[1] and len(down_shape) == 3 and down_shape[2] == w_shape[1]
            and up.shape == (down_shape[0], w_shape[0], down_shape[1]) and ids.dim() == 1 and offsets.shape == (ids.shape[0] + 1,)
            and weight.get_device() == down.get_device() == up.get_device() == offsets.get_device() == ids.get_device() == index
            and (bias is None or (bias.dtype is half and bias.shape == w_shape[:1] and bias.get_device() == index))
            and (residual is None or (residual.dtype is half and residual.shape == (*x_shape[:-1], w_shape[0]) and residual.get_device() == index))):
        _refuse_adapters(name, x, weight, bias, residual, down, up, offsets, ids, dtype)
    N, K = w_shape
    operands = (_aligned(x), _aligned(weight), bias if bias is None else bias.contiguous(), residual if residual is None else _aligned(residual),
                _aligned(down), _aligned(up), offsets.contiguous(), ids.contiguous())
    return index, (x.numel() // K if K else 0, N, K, ids.shape[0], down_shape[0], down_shape[1]), operands


@torch.library.custom_op("fry::adapter_linear", mutates_args=())
def adapter_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor | None, down: torch.Tensor,
                   up: torch.Tensor, offsets: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
    """A linear with a low-rank adapter for each request's rows (the op fry::adapter_linear), fp16:
    x W^T + bias + residual, plus (x down[a]^T) up[a]^T for the rows offsets[s] to offsets[s + 1] of request s, a = ids[s].
    x [..., K], weight [N, K] as nn.Linear holds it, down [adapters, rank, K], up [adapters, N, rank]; offsets [requests + 1]
    and ids [requests] int32 on the device; rows of no request and those of ids -1 have no adapter. rank a multiple of 8 up
    to 128 (pad smaller ones with zeros), N and K multiples of 8. Sums are fp32; from 33 rows on x down^T is rounded to fp16
    between the two products (off by 2^-11 of a value, by 2^-25 below 2^-14; beyond 65504 it stays fp32, which is slower). No
    backward pass."""
    index, shapes, operands = _adapter_operands("adapter_linear", x, weight, bias, residual, down, up, offsets, ids, torch.float16)
    M, N, _, requests, _, rank = shapes
    out = x.new_empty(*x.shape[:-1], N)
    size = _workspace_bytes("fry_adapter_linear_workspace_bytes", M, N, requests, rank)
    workspace = torch.empty(size, device=x.device, dtype=torch.uint8)
    _call(library().fry_adapter_linear, index, *(None if t is None else t.data_ptr() for t in operands), out.data_ptr(), *shapes, workspace.data_ptr(), size)
    return out


@adapter_linear.register_fake
def _(x, weight, bias, residual, down, up, offsets, ids):
    return x.new_empty(*x.shape[:-1], weight.shape[0])


@torch.library.custom_op("fry::int8_adapter_linear", mutates_args=())
def int8_adapter_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None,
                        residual: torch.Tensor | None, down: torch.Tensor, up: torch.Tensor, offsets: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
    """adapter_linear beside the int8 linear (the op fry::int8_adapter_linear): x int8 [..., K] with x_scale fp32 a row,
    weight int8 [N, K] with weight_scale fp32 a row, as int8_linear takes them; the adapters fp16, on the rows that x and
    x_scale stand for. K a multiple of 16."""
    name = "int8_adapter_linear"
    index, shapes, (x, weight, *others) = _adapter_operands(name, x, weight, bias, residual, down, up, offsets, ids, torch.int8)
    M, N, _, requests, _, rank = shapes
    if not (x_scale.dtype is weight_scale.dtype is torch.float32 and x_scale.numel() == M and weight_scale.numel() == N
            and x_scale.get_device() == weight_scale.get_device() == index):
        raise FryError(f"{name} takes an fp32 scale a row of x and of weight on {x.device}, got {x_scale.dtype} {tuple(x_scale.shape)} on "
                       f"{x_scale.device} and {weight_scale.dtype} {tuple(weight_scale.shape)} on {weight_scale.device}")
    x_scale, weight_scale = x_scale.contiguous(), weight_scale.contiguous()
    out = x.new_empty(*x.shape[:-1], N, dtype=torch.float16)
    size = _workspace_bytes("fry_int8_adapter_linear_workspace_bytes", M, N, requests, rank)
    workspace = torch.empty(size, device=x.device, dtype=torch.uint8)
    _call(library().fry_int8_adapter_linear, index, x.data_ptr(), x_scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(),
          *(None if t is None else t.data_ptr() for t in others), out.data_ptr(), *shapes, workspace.data_ptr(), size)
    return out


@int8_adapter_linear.register_fake
def _(x, x_scale, weight, weight_scale, bias, residual, down, up, offsets, ids):
    return x.new_empty(*x.shape[:-1], weight.shape[0], dtype=torch.float16)


@torch.library.custom_op("fry::norm_quant", mutates_args=())
def norm_quant(x: torch.Tensor, gain: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """`chess::norm_quant` (model/int8_blocks.py:191-193): int8 rows of RMSNorm(x) * gain and their scales."""
    _cuda("norm_quant", x, gain)
    _dtype("norm_quant", x, torch.float16, "x")
    x = x.contiguous()
    D = x.shape[-1]
    q = torch.empty(x.shape, device=x.device, dtype=torch.int8)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    library().fry_norm_quant(_ptr(x), _ptr(gain.contiguous()), eps, _ptr(q), _ptr(scale), x.numel() // D, D, _stream(x))
    return q, scale


@norm_quant.register_fake
def _(x, gain, eps):
    return x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("fry::mix_norm_quant", mutates_args=())
def mix_norm_quant(x: torch.Tensor, original: torch.Tensor, residual_scale: torch.Tensor, input_scale: torch.Tensor, gain: torch.Tensor,
                   eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """`chess::mix_norm_quant` (model/int8_blocks.py:201-207): the block input mixed with the embedding, then norm_quant."""
    _cuda("mix_norm_quant", x, original, residual_scale, input_scale, gain)
    x, original = x.contiguous(), original.contiguous()
    D = x.shape[-1]
    mixed = torch.empty_like(x, dtype=torch.float16)
    q = torch.empty(x.shape, device=x.device, dtype=torch.int8)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    library().fry_mix_norm_quant(_ptr(x), _ptr(original), _ptr(residual_scale), _ptr(input_scale), _ptr(gain.contiguous()), eps,
                                 _ptr(mixed), _ptr(q), _ptr(scale), x.numel() // D, D, _stream(x))
    return mixed, q, scale


@mix_norm_quant.register_fake
def _(x, original, residual_scale, input_scale, gain, eps):
    return x.new_empty(x.shape, dtype=torch.float16), x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("fry::rotate_quant", mutates_args=())
def rotate_quant(h: torch.Tensor, hadamard_signs: torch.Tensor, width: int) -> tuple[torch.Tensor, torch.Tensor]:
    """`chess::rotate_quant` (model/int8_blocks.py:234-246). The kernel applies Sylvester's 32x32 signs itself, the matrix
    the reference passes as hadamard_signs (`hadamard(32)`, model/int8_blocks.py:54-58); any other matrix is refused."""
    _cuda("rotate_quant", h)
    if tuple(hadamard_signs.shape) != (HADAMARD_BLOCK, HADAMARD_BLOCK):
        raise FryError(f"rotate_quant rotates by 32x32 Hadamard blocks, got signs of shape {tuple(hadamard_signs.shape)}")
    h = h.contiguous()
    hidden = h.shape[-1]
    q = torch.empty(*h.shape[:-1], width, device=h.device, dtype=torch.int8)
    scale = torch.empty(h.shape[:-1], device=h.device, dtype=torch.float32)
    library().fry_rotate_quant(_ptr(h), _ptr(q), _ptr(scale), h.numel() // hidden, hidden, width, _stream(h))
    return q, scale


@rotate_quant.register_fake
def _(h, hadamard_signs, width):
    return h.new_empty(*h.shape[:-1], width, dtype=torch.int8), h.new_empty(h.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("fry::template_attention", mutates_args=())
def template_attention(projected: torch.Tensor, templates: torch.Tensor, q_gain: torch.Tensor, k_gain: torch.Tensor, heads: int,
                       kv_heads: int, dq: int, dv: int, templates_count: int, eps: float) -> torch.Tensor:
    """`chess::template_attention` (model/fused_blocks.py:104-171): projected [B, 70, q|k|v|mix] -> [B, 70, heads * dv]."""
    _cuda("template_attention", projected, templates, q_gain, k_gain)
    projected = projected.contiguous()
    B, T, _ = projected.shape
    if T != 70:
        raise FryError(f"template_attention takes 70 tokens a position, got {T}")
    out = projected.new_empty(B, T, heads * dv)
    paired = pair_templates(templates)
    library().fry_template_attention(_ptr(projected), _ptr(paired), _ptr(q_gain.contiguous()), _ptr(k_gain.contiguous()),
                                     _ptr(out), B, heads, kv_heads, dq, dv, templates_count, eps, _stream(projected))
    return out


def pair_templates(templates: torch.Tensor) -> torch.Tensor:
    """The templates [8, 64, 64] re-laid as [64, 64, 8] for the attention kernel (the reference's `paired_templates`,
    model/attention_cuda.py:412-434). Paired afresh on every call here, on the current stream, so that the op records
    into CUDA graphs; the network pairs its templates once."""
    _cuda("pair_templates", templates)
    if tuple(templates.shape) != (8, 64, 64) or templates.dtype != torch.float16:
        raise FryError(f"the attention takes 8 fp16 templates of 64 x 64, got {tuple(templates.shape)} {templates.dtype}")
    templates = templates.contiguous()
    paired = templates.new_empty(64, 64, 8)
    library().fry_pair_templates(_ptr(templates), _ptr(paired), 8, _stream(templates))
    return paired


@template_attention.register_fake
def _(projected, templates, q_gain, k_gain, heads, kv_heads, dq, dv, templates_count, eps):
    B, T, _ = projected.shape
    return projected.new_empty(B, T, heads * dv)


@torch.library.custom_op("fry::linear", mutates_args=())
def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
           gated: bool = False, accumulate_fp32: bool = False, original: torch.Tensor | None = None,
           residual_scale: torch.Tensor | None = None, input_scale: torch.Tensor | None = None) -> torch.Tensor:
    """`chess::linear` (model/fused_blocks.py:308-313) for fp16 x and weight [K, N] as the reference stores it ([K, 2N],
    gate columns then up columns, gated): fp32 accumulation (the reference accumulates fp16 inputs in fp16 unless
    accumulate_fp32), fp16 out, or fp32 out with accumulate_fp32; the gated and input-mixing forms (the fp16 blocks')
    in fp16."""
    _cuda("linear", x, weight, bias, residual, original, residual_scale, input_scale)
    _dtype("linear", x, torch.float16, "x")
    if gated or original is not None:  # the fp16 blocks' forms (fp16 out)
        if accumulate_fp32:
            raise FryError("fry::linear gives its gated and input-mixing forms in fp16 only")
        K, width = weight.shape
        N = width // 2 if gated else width
        x = x.contiguous()
        M = x.numel() // K
        out = x.new_empty(*x.shape[:-1], N, dtype=torch.float16)
        bias = bias.half().contiguous() if bias is not None else None
        residual = residual.contiguous() if residual is not None else None
        original = original.contiguous() if original is not None else None
        library().fry_linear_full(_ptr(x), _ptr(weight.t().contiguous()), _ptr(bias), _ptr(residual), _ptr(original), _ptr(residual_scale),
                                  _ptr(input_scale), _ptr(out), M, N, K, int(gated), _stream(x))
        return out
    K, N = weight.shape
    x = x.contiguous()
    M = x.numel() // K
    out = x.new_empty(*x.shape[:-1], N, dtype=torch.float32 if accumulate_fp32 else torch.float16)
    if bias is not None:
        bias = bias.float().contiguous() if accumulate_fp32 else bias.half().contiguous()
    weight_nk = weight.t().contiguous()
    residual = residual.contiguous() if residual is not None else None
    library().fry_linear(_ptr(x), _ptr(weight_nk), _ptr(bias), _ptr(residual), _ptr(out), M, N, K, int(accumulate_fp32), _stream(x))
    return out


@linear.register_fake
def _(x, weight, bias=None, residual=None, gated=False, accumulate_fp32=False, original=None, residual_scale=None, input_scale=None):
    return x.new_empty(*x.shape[:-1], weight.shape[1] // 2 if gated else weight.shape[1], dtype=torch.float32 if accumulate_fp32 else x.dtype)


@torch.library.custom_op("fry::linear_norm_quant", mutates_args=())
def linear_norm_quant(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor | None, gain: torch.Tensor,
                      eps: float) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """`chess::linear` (fp16, weight [K, N] as the reference stores it) then `chess::norm_quant` of its output
    (model/int8_blocks.py:191-193, 274-288) as one kernel: (out, q, scale). out equals `linear`'s bit for bit; q and scale
    equal `norm_quant(out, gain, eps)` to within its rounding. N a multiple of 256 up to 1024."""
    _cuda("linear_norm_quant", x, weight, bias, residual, gain)
    _dtype("linear_norm_quant", x, torch.float16, "x")
    K, N = weight.shape
    x = x.contiguous()
    M = x.numel() // K
    out = x.new_empty(*x.shape[:-1], N, dtype=torch.float16)
    q = x.new_empty(*x.shape[:-1], N, dtype=torch.int8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    bias = bias.half().contiguous() if bias is not None else None
    residual = residual.contiguous() if residual is not None else None
    library().fry_linear_norm_quant(_ptr(x), _ptr(weight.t().contiguous()), _ptr(bias), _ptr(residual), _ptr(out), _ptr(gain.half().contiguous()),
                                    eps, _ptr(q), _ptr(scale), M, N, K, _stream(x))
    return out, q, scale


@linear_norm_quant.register_fake
def _(x, weight, bias, residual, gain, eps):
    shape = (*x.shape[:-1], weight.shape[1])
    return x.new_empty(shape, dtype=torch.float16), x.new_empty(shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)


@torch.library.custom_op("fry::board_embedding", mutates_args=())
def board_embedding(boards: torch.Tensor, embed: torch.Tensor, position: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """`chess::board_embedding` (model/fused_blocks.py:495-507): boards [B, 70] -> [B, 70, D] fp16, the 23 square-feature
    rows of `SquareFeatures.indices` found in the kernel (the reference's rays and jumps tables are built in)."""
    _cuda("board_embedding", boards, embed, position, table)
    boards = boards.long().contiguous()
    B, T = boards.shape
    D = table.shape[1]
    out = table.new_empty(B, T, D)
    library().fry_board_embedding(_ptr(boards), _ptr(embed.contiguous()), _ptr(position.contiguous()), _ptr(table.contiguous()), _ptr(out),
                                  B, D, _stream(boards))
    return out


@board_embedding.register_fake
def _(boards, embed, position, table):
    return table.new_empty(*boards.shape, table.shape[1])


def heads_struct(ln_gain, a_weight, a_bias, narrow_weight, narrow_bias, hidden_weight, hidden_bias, out_weight, out_bias) -> FryHeads:
    return FryHeads(_ptr(ln_gain), _ptr(a_weight), _ptr(a_bias), _ptr(narrow_weight), _ptr(narrow_bias), _ptr(hidden_weight),
                    _ptr(hidden_bias), _ptr(out_weight), _ptr(out_bias), out_weight.shape[0])


@torch.library.custom_op("fry::heads", mutates_args=())
def heads(stream: torch.Tensor, ln_gain: torch.Tensor, a_weight: torch.Tensor, a_bias: torch.Tensor, narrow_weight: torch.Tensor,
          narrow_bias: torch.Tensor, hidden_weight: torch.Tensor, hidden_bias: torch.Tensor, out_weight: torch.Tensor,
          out_bias: torch.Tensor, eps: float) -> torch.Tensor:
    """The heads from the last block's stream to the answer rows [B, 1969] (the reference's `heads` op,
    model/fused_blocks.py:743-774, computes the same rows from its own folded weights). a_weight is [N, K] fp16:
    (W_f^T W_t / sqrt d)^T; narrow_weight [21, d] fp32; the eval head's layers as nn.Linear holds them, in fp32."""
    _cuda("heads", stream, ln_gain, a_weight, a_bias, narrow_weight, narrow_bias, hidden_weight, hidden_bias, out_weight, out_bias)
    stream = stream.contiguous()
    B, T, D = stream.shape
    rows = torch.empty(B, 1969, device=stream.device, dtype=torch.float32)
    lib = library()
    workspace = torch.empty(lib.fry_heads_workspace_bytes(B, D), device=stream.device, dtype=torch.uint8)
    weights = heads_struct(ln_gain, a_weight, a_bias, narrow_weight, narrow_bias, hidden_weight, hidden_bias, out_weight, out_bias)
    lib.fry_heads(_ptr(stream), ctypes.byref(weights), eps, _ptr(rows), _ptr(workspace), workspace.numel(), B, D, _stream(stream))
    return rows


@heads.register_fake
def _(stream, ln_gain, a_weight, a_bias, narrow_weight, narrow_bias, hidden_weight, hidden_bias, out_weight, out_bias, eps):
    return stream.new_empty(stream.shape[0], 1969, dtype=torch.float32)
