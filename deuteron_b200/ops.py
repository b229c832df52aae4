"""Device-resident operators: thin wrappers that hand torch CUDA tensors' pointers to the C ABI.

torch is used for device memory and streams only; every computation below runs in
libdeuteron_b200.so on the current torch stream. Tensors must live on the current CUDA device.
"""
from __future__ import annotations

import ctypes as ct
import math

import torch

from . import native


_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)   # the handle alone: 0.3 us where the Stream object takes 3.2


def _stream() -> int:
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


def _require_cuda(*tensors: torch.Tensor) -> None:
    for tensor in tensors:
        if not isinstance(tensor, torch.Tensor) or not tensor.is_cuda:
            raise ValueError('deuteron_b200 operators take CUDA tensors')


def _flat(tensor: torch.Tensor, dtype: torch.dtype, label: str) -> torch.Tensor:
    if tensor.dtype != dtype:
        raise ValueError(f'{label} must have dtype {dtype}, got {tensor.dtype}')
    if not tensor.is_contiguous():
        raise ValueError(f'{label} must be contiguous')
    return tensor


# ------------------------------------------------------------------------------------------------
# elementwise / f16
# ------------------------------------------------------------------------------------------------


def elementwise(op: str, x: torch.Tensor, y: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """out = op(x, y) or op(x) elementwise in FP32 (operator names of the reference's ElementwiseImpl)."""
    if op not in native.ELEMENTWISE_OPS:
        raise NotImplementedError(f'elementwise operation {op}')
    binary = op in native.BINARY_OPS
    _require_cuda(x)
    _flat(x, torch.float32, 'x')
    if binary:
        if y is None:
            raise ValueError(f'{op} needs two operands')
        _require_cuda(y)
        _flat(y, torch.float32, 'y')
        if y.shape != x.shape:
            raise ValueError('operand shapes differ')
    if out is None:
        out = torch.empty_like(x)
    _require_cuda(out)
    _flat(out, torch.float32, 'out')
    if out.shape != x.shape:
        raise ValueError('output shape differs')
    native.call('dtn_elementwise_f32', native.ELEMENTWISE_OPS[op], x.data_ptr(), y.data_ptr() if binary else None,
                out.data_ptr(), x.numel(), _stream())
    return out


def add(x: torch.Tensor, y: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    return elementwise('add', x, y, out)


def f16_copy(src: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _require_cuda(src)
    _flat(src, torch.float16, 'src')
    out = torch.empty_like(src) if out is None else _flat(out, torch.float16, 'out')
    native.call('dtn_f16_copy', src.data_ptr(), out.data_ptr(), src.numel(), _stream())
    return out


def f16_widen(src: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _require_cuda(src)
    _flat(src, torch.float16, 'src')
    out = torch.empty(src.shape, dtype=torch.float32, device=src.device) if out is None else _flat(out, torch.float32, 'out')
    native.call('dtn_f16_widen', src.data_ptr(), out.data_ptr(), src.numel(), _stream())
    return out


def f16_narrow(src: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    _require_cuda(src)
    _flat(src, torch.float32, 'src')
    out = torch.empty(src.shape, dtype=torch.float16, device=src.device) if out is None else _flat(out, torch.float16, 'out')
    native.call('dtn_f16_narrow', src.data_ptr(), out.data_ptr(), src.numel(), _stream())
    return out


# ------------------------------------------------------------------------------------------------
# row reductions
# ------------------------------------------------------------------------------------------------


def row_reduce(op: str, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r] = sum / max / sumsq of row r of the 2-D FP32 tensor x (rows may be strided)."""
    if op not in ('sum', 'max', 'sumsq'):
        raise NotImplementedError(f'row reduction {op}')
    _require_cuda(x)
    if x.dtype != torch.float32 or x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError('row_reduce takes a 2-D float32 tensor with unit column stride')
    rows, cols = x.shape
    ldx = x.stride(0) if rows > 1 else max(cols, 1)
    if out is None:
        out = torch.empty(rows, dtype=torch.float32, device=x.device)
    _flat(out, torch.float32, 'out')
    native.call('dtn_row_reduce_f32', native.REDUCE_OPS[op], x.data_ptr(), out.data_ptr(), rows, cols, max(ldx, cols), _stream())
    return out


def _row_matrix(x: torch.Tensor, label: str) -> tuple[int, int, int]:
    _require_cuda(x)
    if x.dtype != torch.float32 or x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f'{label} takes a 2-D float32 tensor with unit column stride')
    rows, cols = x.shape
    return rows, cols, max(x.stride(0) if rows > 1 else cols, cols, 1)


def _row_fused(reduce: str, x: torch.Tensor, program: list[tuple[str, int, int, int]], n_scalar: int, out_reg: int, inputs=(),
               per_row: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """One launch of the fused row kernel. program: (operator, destination, a, b) over the registers
    0 = reduced value, 1 = sum of exponentials, 2 = row element, 3 + i = inputs[i]; inputs: a float
    (immediate), a one-element tensor (scalar) or a tensor of `cols` values (one per column)."""
    rows, cols, ldx = _row_matrix(x, 'row kernel')
    described, pointers = [], []
    for item in inputs:
        if isinstance(item, (int, float)):
            described.append({'kind': 'immediate', 'value': float(item)})
            pointers.append(None)
            continue
        _flat(item, torch.float32, 'row kernel input')
        if item.numel() not in (1, cols):
            raise ValueError('row kernel inputs hold one value or one value per column')
        described.append({'kind': 'columns' if item.numel() == cols and cols != 1 else 'scalar'})
        pointers.append(item.data_ptr())
    if out is None:
        out = torch.empty(rows if per_row else (rows, cols), dtype=torch.float32, device=x.device)
    _flat(out, torch.float32, 'out')
    params = {'reduce': reduce, 'rows': rows, 'cols': cols, 'inputs': described, 'n_scalar': n_scalar, 'out_reg': out_reg,
              'ops': [native.ELEMENTWISE_OPS[p[0]] for p in program], 'dst': [p[1] for p in program],
              'a': [p[2] for p in program], 'b': [p[3] for p in program], 'per_row': per_row}
    if not _row_specialized(params, x, pointers, out, ldx):
        native.row_fused(params, x.data_ptr(), pointers, out.data_ptr(), ldx, 0 if per_row else max(cols, 1), _stream())
    return out


_row_kernels: dict[tuple, tuple | None] = {}


def _row_specialized(params: dict, x: torch.Tensor, pointers: list, out: torch.Tensor, ldx: int) -> bool:
    """Runs the kernel written for this one program (jit.py) when there is one: dense rows, 16-byte aligned buffers.
    With no program to decode and a row's loads all requested up front it is the faster kernel at every size it
    takes; False sends the launch to the library's kernel."""
    from . import jit
    addresses = [x.data_ptr(), out.data_ptr(), *[p for p in pointers if p is not None]]
    if not jit.enabled() or ldx != params['cols'] or params['rows'] == 0 or any(a % 16 for a in addresses):
        return False
    device = x.device.index if x.device.index is not None else torch.cuda.current_device()
    key = (device, repr(sorted(params.items())))
    if key not in _row_kernels:
        if torch.cuda.is_current_stream_capturing():   # a module is not loaded inside a capture: the library kernel this once
            return False
        buffers = {'x': ('x', 0), 'out': ('out', 0), **{f'in{i}': (f'in{i}', 0) for i in range(len(pointers))}}
        spec = jit.row_source(params, buffers)
        kernel = jit.kernel_for(spec, device) if spec is not None else None
        _row_kernels[key] = (spec, kernel) if kernel is not None else None
    entry = _row_kernels[key]
    if entry is None:
        return False
    roles = {'x': x.data_ptr(), 'out': out.data_ptr(), **{f'in{i}': p for i, p in enumerate(pointers)}}
    jit.launch(entry[0], entry[1], roles.__getitem__, _stream())
    return True


def row_softmax(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r, c] = exp(x[r, c] - max_r) / sum_c exp(x[r, c] - max_r), one launch."""
    return _row_fused('softmax', x, [('reciprocal', 3, 1, 1), ('subtract', 4, 2, 0), ('exp', 4, 4, 4), ('multiply', 4, 4, 3)], 1, 4, out=out)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, epsilon: float = 1e-5, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r, c] = x[r, c] * rsqrt(mean_c(x[r, :]^2) + epsilon) * weight[c], one launch."""
    program = [('divide', 6, 0, 4), ('add', 6, 6, 5), ('rsqrt', 6, 6, 6), ('multiply', 7, 2, 6), ('multiply', 7, 7, 3)]
    return _row_fused('sumsq', x, program, 3, 7, inputs=(weight, float(x.shape[1]), float(epsilon)), out=out)


def l2_norm(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r, c] = x[r, c] * rsqrt(sum_c x[r, :]^2), one launch."""
    return _row_fused('sumsq', x, [('rsqrt', 3, 0, 0), ('multiply', 4, 2, 3)], 1, 4, out=out)


def row_mean(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r] = sum_c x[r, c] / cols, one launch."""
    return _row_fused('sum', x, [('divide', 4, 0, 3)], 1, 4, inputs=(float(x.shape[1]),), per_row=True, out=out)


# ------------------------------------------------------------------------------------------------
# GEMM
# ------------------------------------------------------------------------------------------------

_workspaces: dict[tuple[int, int], torch.Tensor] = {}


def gemm_workspace_bytes(mode: str, m: int, n: int, k: int) -> int:
    size = ct.c_size_t(0)
    native.call('dtn_gemm_workspace_bytes', native.GEMM_MODES[mode], m, n, k, ct.byref(size))
    return size.value


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    """Scratch for the operand planes, cached per (device, stream) and grown on demand."""
    key = (device.index if device.index is not None else torch.cuda.current_device(), _stream())
    buffer = _workspaces.get(key)
    if buffer is None or buffer.numel() < nbytes + 1024:
        buffer = torch.empty(nbytes + 1024, dtype=torch.uint8, device=device)
        _workspaces[key] = buffer
    return buffer


def _row_major(tensor: torch.Tensor, label: str) -> int:
    if tensor.dtype != torch.float32 or tensor.dim() != 2:
        raise ValueError(f'{label} must be a 2-D float32 tensor')
    if tensor.shape[1] > 1 and tensor.stride(1) != 1:
        raise ValueError(f'{label} must be row-major (unit column stride)')
    return tensor.stride(0) if tensor.shape[0] > 1 else max(tensor.shape[1], 1)


def gemm(a: torch.Tensor, b: torch.Tensor, mode: str = 'bf16x3', out: torch.Tensor | None = None,
         workspace: torch.Tensor | None = None, phase: int = 3) -> torch.Tensor:
    """C = A @ B with FP32 storage and the reference's contraction_precision `mode`.

    a[M,K], b[K,N], out[M,N]: row-major; rows may be strided (a column block of a wider matrix).
    `phase` 1 runs only the operand split into the workspace, 2 only the product kernel on planes
    already there, 3 (default) both.
    """
    if mode not in native.GEMM_MODES:
        raise ValueError(f'unsupported contraction precision {mode!r}')
    _require_cuda(a, b)
    lda, ldb = _row_major(a, 'a'), _row_major(b, 'b')
    m, k = a.shape
    k2, n = b.shape
    if k != k2:
        raise ValueError(f'inner dimensions differ: {k} vs {k2}')
    if out is None:
        out = torch.empty((m, n), dtype=torch.float32, device=a.device)
    _require_cuda(out)
    ldc = _row_major(out, 'out')
    if tuple(out.shape) != (m, n):
        raise ValueError('output shape differs')
    nbytes = gemm_workspace_bytes(mode, m, n, k)
    ws_ptr, ws_bytes = None, 0
    if nbytes:
        if workspace is None:
            workspace = _workspace(nbytes, a.device)
        base = workspace.data_ptr()
        ws_ptr = (base + 1023) // 1024 * 1024
        ws_bytes = workspace.numel() * workspace.element_size() - (ws_ptr - base)
    native.call('dtn_gemm_x3_phase', native.GEMM_MODES[mode], a.data_ptr(), b.data_ptr(), out.data_ptr(), m, n, k,
                max(lda, k), max(ldb, n), max(ldc, n), ws_ptr, ws_bytes, phase, _stream())
    return out


def push_block(src: torch.Tensor, destinations: list[torch.Tensor]) -> None:
    """Writes the 2-D float32 block `src` into every tensor of `destinations` (same shape, equal row strides; up to
    seven; they may be views of other GPUs' memory) with one kernel that reads the block once."""
    _require_cuda(src)
    lds = _row_major(src, 'src')
    if not destinations:
        return
    rows, cols = src.shape
    strides = set()
    for dst in destinations:
        if dst.dtype != torch.float32 or tuple(dst.shape) != (rows, cols):
            raise ValueError('every destination must be a float32 tensor of the shape of src')
        strides.add(_row_major(dst, 'destination'))
    if len(strides) != 1:
        raise ValueError('the destinations must share one row stride')
    pointers = (ct.c_void_p * len(destinations))(*[dst.data_ptr() for dst in destinations])
    native.call('dtn_push_block', src.data_ptr(), max(lds, cols), pointers, len(destinations), max(strides.pop(), cols), rows, cols,
                _stream())


def set_gemm_variant(variant: int) -> None:
    native.call('dtn_gemm_set_variant', variant)


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------


def attention(q: torch.Tensor, kt: torch.Tensor, v: torch.Tensor, scale: float, out: torch.Tensor | None = None) -> torch.Tensor:
    """Single-head attention in the reference's example layout: q[rows,depth], kt[depth,keys], v[keys,cols]."""
    _require_cuda(q, kt, v)
    for tensor, label in ((q, 'q'), (kt, 'kt'), (v, 'v')):
        _flat(tensor, torch.float32, label)
        if tensor.dim() != 2:
            raise ValueError(f'{label} must be 2-D')
    rows, depth = q.shape
    depth2, keys = kt.shape
    keys2, cols = v.shape
    if depth != depth2 or keys != keys2:
        raise ValueError('attention operand shapes disagree')
    if out is None:
        out = torch.empty((rows, cols), dtype=torch.float32, device=q.device)
    _flat(out, torch.float32, 'out')
    native.call('dtn_attention_f32', q.data_ptr(), kt.data_ptr(), v.data_ptr(), out.data_ptr(), rows, keys, depth, cols,
                float(scale), _stream())
    return out


def gqa_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, out: torch.Tensor | None = None,
                  groups: tuple[int, int] | None = None) -> torch.Tensor:
    """Grouped-query attention forward, non-causal: q[B,Hq,S,D], k/v[B,Hkv,S,D] (f16 or f32) -> out[B,Hq,S,D] f32.

    `groups=(begin, end)` restricts the computation to that range of the B*Hkv (batch, kv-head) groups.
    """
    _require_cuda(q, k, v)
    if q.dtype not in (torch.float16, torch.float32) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError('q, k, v must share dtype float16 or float32')
    for tensor, label in ((q, 'q'), (k, 'k'), (v, 'v')):
        if tensor.dim() != 4 or not tensor.is_contiguous():
            raise ValueError(f'{label} must be a contiguous [B,H,S,D] tensor')
    b, hq, s, d = q.shape
    if k.shape != v.shape or k.shape[0] != b or k.shape[2] != s or k.shape[3] != d:
        raise ValueError('k/v shapes disagree with q')
    hkv = k.shape[1]
    if out is None:
        out = torch.empty((b, hq, s, d), dtype=torch.float32, device=q.device)
    _flat(out, torch.float32, 'out')
    begin, end = groups if groups is not None else (0, b * hkv)
    native.call('dtn_gqa_fwd', q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), b, hq, hkv, s, d, float(scale),
                native.STORAGE['f16' if q.dtype == torch.float16 else 'f32'], begin, end, _stream())
    return out


def set_gqa_variant(variant: int) -> None:
    native.call('dtn_gqa_set_variant', variant)


# ------------------------------------------------------------------------------------------------
# rotary positions and the paged key-value cache
# ------------------------------------------------------------------------------------------------

_STORAGE_OF = {torch.float32: native.STORAGE['f32'], torch.float16: native.STORAGE['f16'], torch.bfloat16: native.STORAGE['bf16']}
_LAYOUTS = {'half': 0, 'interleaved': 1}


def _on_current_device(*tensors: torch.Tensor) -> None:
    current = torch.cuda.current_device() if tensors[0].is_cuda else None
    for tensor in tensors:   # -1 for a tensor of the CPU
        if tensor.get_device() != current:
            if not tensor.is_cuda:
                raise ValueError('deuteron_b200 operators take CUDA tensors')
            raise ValueError(f'a tensor is on {tensor.device}, the current device is {torch.cuda.current_device()}')


def _tensors(*tensors: torch.Tensor) -> None:
    for tensor in tensors:
        if not isinstance(tensor, torch.Tensor):
            raise ValueError(f'a tensor is needed, got {type(tensor).__name__}')


def _heads(tensor: torch.Tensor, label: str, written: bool = False) -> tuple[int, int]:
    """Token and head strides of a [tokens, heads, dim] tensor with dense heads (0 for an extent of one)."""
    shape = tensor.shape
    if len(shape) != 3:
        raise ValueError(f'{label} must be a [tokens, heads, dim] tensor')
    tokens, heads, dim = shape
    if tensor.is_contiguous():
        return heads * dim if tokens > 1 else 0, dim if heads > 1 else 0
    token_stride, head_stride, unit = tensor.stride()
    if dim > 1 and unit != 1:
        raise ValueError(f'{label} must have dense heads (unit stride in its last dimension)')
    token_stride, head_stride = token_stride if tokens > 1 else 0, head_stride if heads > 1 else 0
    if written and ((tokens > 1 and token_stride == 0) or (heads > 1 and head_stride == 0)):
        raise ValueError(f'{label} must not be an expanded tensor: it is written')
    return token_stride, head_stride


def _index(tensor: torch.Tensor, label: str, count: int | None = None, wide: bool = False) -> None:
    dtype, shape = tensor.dtype, tensor.shape
    if len(shape) != 1 or not tensor.is_contiguous():
        raise ValueError(f'{label} must be a contiguous 1-D tensor')
    if dtype is not torch.int32 and not (wide and dtype is torch.int64):
        raise ValueError(f'{label} must have dtype {"int32 or int64" if wide else "int32"}, got {dtype}')
    if count is not None and shape[0] != count:
        raise ValueError(f'{label} must have {count} entries, got {shape[0]}')


def _rotation(frequencies: torch.Tensor | None, layout: str, dim: int) -> int:
    """Number of rotated pairs; checks frequencies and layout."""
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    if frequencies is None:
        return 0
    if not isinstance(frequencies, torch.Tensor) or frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous():
        raise ValueError('frequencies must be a contiguous 1-D float64 tensor (radians per position)')
    pairs = frequencies.shape[0]
    if 2 * pairs > dim:
        raise ValueError(f'{pairs} frequencies rotate {2 * pairs} elements, a head has {dim}')
    return pairs


def _pools(k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor) -> tuple[int, int, int, int, int, int, int, int, int]:
    """Pages, kv heads, page size, head size, page and head strides of both pools, then sequences, pages per sequence and row
    stride of the tables, all checked."""
    shape = k_pages.shape
    if len(shape) != 4 or v_pages.dim() != 4:
        raise ValueError(f'{"k_pages" if len(shape) != 4 else "v_pages"} must be a [pages, kv_heads, page_size, dim] tensor')
    if shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError('k_pages and v_pages must have one shape and dtype')
    pages, heads, size, dim = shape
    if size < 1:
        raise ValueError('a page holds at least one token')
    if k_pages.is_contiguous() and v_pages.is_contiguous():
        head = size * dim
        page = heads * head
    else:
        strides = k_pages.stride()
        page, head, token, unit = strides
        if (dim > 1 and unit != 1) or (size > 1 and token != dim):
            raise ValueError('the rows of one page and head must be dense in k_pages and v_pages')
        if strides != v_pages.stride():   # strides of extents of one are nobody's business
            if any(extent > 1 and a != b for extent, a, b in zip(shape, strides, v_pages.stride())):
                raise ValueError('k_pages and v_pages must have the same strides')
    if tables.dtype != torch.int32 or tables.dim() != 2:
        raise ValueError('tables must be a [sequences, pages per sequence] int32 tensor')
    sequences, width = tables.shape
    row, column = tables.stride()
    if width > 1 and column != 1:
        raise ValueError('tables must have unit column stride')
    return pages, heads, size, dim, page if pages > 1 else 0, head if heads > 1 else 0, sequences, width, row if sequences > 1 else 0


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str | None = None, factor: float = 1.0,
                       original_length: int | None = None, fast: float = 32.0, slow: float = 1.0,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """Frequencies (float64, radians per position, one per pair of `rotary_dim` elements) and amplitude for `rotary`.

    w_i = base^(-2i / rotary_dim). `scaling` stretches them for contexts `factor` times longer than trained: 'linear'
    divides every frequency by the factor; 'ntk' raises the base by factor^(rotary_dim / (rotary_dim - 2)), which leaves the
    first pair alone and divides the last by the factor; 'yarn' (Peng et al., 2023) divides those that turn fewer than `slow`
    times within `original_length`, keeps those that turn more than `fast` times, blends in between by the number of
    turns, and returns the amplitude 0.1 ln(factor) + 1. (Some published models blend linearly in the pair's index between the two
    bounds, or take another amplitude: their middle pairs differ. Any float64 tensor of frequencies can be passed to `rotary`
    instead.) `device` defaults to the current CUDA device.
    """
    if type(rotary_dim) is not int or rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f'rotary_dim must be an even non-negative integer, got {rotary_dim!r}')
    if not (base > 0 and factor > 0) or base == float('inf') or factor == float('inf'):
        raise ValueError('base and factor must be positive and finite')
    if scaling not in (None, 'linear', 'ntk', 'yarn'):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    if scaling is None and factor != 1.0:
        raise ValueError('a factor needs a scaling')
    amplitude = 1.0
    if scaling == 'ntk':
        if rotary_dim == 2:
            raise ValueError("'ntk' needs more than one pair")
        base = base * factor ** (rotary_dim / (rotary_dim - 2)) if rotary_dim else base
    frequencies = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling == 'linear':
        frequencies = [w / factor for w in frequencies]
    if scaling == 'yarn':
        if not original_length or original_length < 1 or not 0 <= slow < fast:
            raise ValueError("'yarn' needs the original_length of training and 0 <= slow < fast")
        kept = [min(max((original_length * w / (2 * math.pi) - slow) / (fast - slow), 0.0), 1.0) for w in frequencies]
        frequencies = [w * keep + w / factor * (1.0 - keep) for w, keep in zip(frequencies, kept)]
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return torch.tensor(frequencies, dtype=torch.float64, device='cuda' if device is None else device), amplitude


class _Turned(torch.autograd.Function):
    """`rotary` and `rotary_backward` where a gradient is recorded: each is the other's."""

    @staticmethod
    def forward(ctx, x, positions, frequencies, layout, amplitude, transpose):
        ctx.save_for_backward(positions, frequencies)
        ctx.rest = layout, amplitude, 1 - transpose
        return _rotary(x, positions, frequencies, layout, amplitude, None, transpose)

    @staticmethod
    def backward(ctx, grad):
        if grad.shape[-1] > 1 and grad.stride(-1) != 1:   # a sum's gradient is one value expanded
            grad = grad.contiguous()
        return _rotary(grad, *ctx.saved_tensors, *ctx.rest[:2], None, ctx.rest[2]), None, None, None, None, None


def _rotary(x, positions, frequencies, layout, amplitude, out, transpose) -> torch.Tensor:
    _tensors(x, positions, frequencies)
    if (x.requires_grad or frequencies.requires_grad) and torch.is_grad_enabled():
        if frequencies.requires_grad:
            raise ValueError('frequencies have no gradient')
        if out is not None:
            raise ValueError('a result in `out` has no gradient: call without it, or under torch.no_grad()')
        return _Turned.apply(x, positions, frequencies, layout, amplitude, transpose)
    if x.dtype not in _STORAGE_OF:
        raise ValueError(f'x must have dtype float32, float16 or bfloat16, got {x.dtype}')
    token_stride, head_stride = _heads(x, 'x')
    tokens, heads, dim = x.shape
    _index(positions, 'positions', tokens, wide=True)
    pairs = _rotation(frequencies, layout, dim)
    if out is None:
        _on_current_device(x, positions, frequencies)
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        out_token_stride, out_head_stride = heads * dim, dim
    else:
        _tensors(out)
        if out.dtype != x.dtype or out.shape != x.shape:
            raise ValueError('out must have the shape and dtype of x')
        out_token_stride, out_head_stride = _heads(out, 'out', written=True)
        if out.data_ptr() == x.data_ptr() and (out_token_stride, out_head_stride) != (token_stride, head_stride):
            raise ValueError('out must be x itself or lie elsewhere')
        _on_current_device(x, positions, frequencies, out)
    native.call('dtn_rotary', native.ROTARY_ARGS.pack(
        x.data_ptr(), out.data_ptr(), positions.data_ptr(), frequencies.data_ptr(), positions.dtype is torch.int64, tokens, heads, dim, pairs,
        token_stride, head_stride, out_token_stride, out_head_stride, _LAYOUTS[layout], transpose, _STORAGE_OF[x.dtype], float(amplitude)), _stream())
    return out


def rotary(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, layout: str = 'half', amplitude: float = 1.0,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary positions: turns pair i of every head of token t by positions[t] * frequencies[i] and scales it by `amplitude`.

    x: [tokens, heads, dim], float32 / float16 / bfloat16, any token and head strides, dense heads (a slice of a fused
    projection); positions: int32 or int64 [tokens]; frequencies: float64 [pairs] from `rotary_frequencies`. Pair i is
    (i, i + pairs) in the 'half' layout, (2i, 2i + 1) in the 'interleaved' one; elements from 2 * pairs on are copied. The
    angle is formed in 64 bits and reduced to a fraction of a turn; its sine and cosine and the rotation are FP32 (2^-21 of a pair's
    magnitude), the result is rounded once. `out` may be x itself; otherwise it must not overlap x. The gradient of x is recorded
    where x requires one (`rotary_backward`); positions and frequencies have none.
    """
    return _rotary(x, positions, frequencies, layout, amplitude, out, 0)


def rotary_backward(grad: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, layout: str = 'half', amplitude: float = 1.0,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Gradient of `rotary`'s x from the gradient of its result: the transposed map (each pair turned back, times `amplitude`).
    Same arguments."""
    return _rotary(grad, positions, frequencies, layout, amplitude, out, 1)


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, rows: torch.Tensor,
                 positions: torch.Tensor, frequencies: torch.Tensor | None = None, layout: str = 'half', amplitude: float = 1.0,
                 q: torch.Tensor | None = None, q_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes the keys and values of new tokens into the pages of a cache; rotates keys and queries on the way. One launch.

    k, v: [tokens, kv_heads, dim]; k_pages, v_pages: [pages, kv_heads, page_size, dim] with equal strides; tables: int32
    [sequences, pages per sequence]. Token t is position positions[t] (int32 or int64) of sequence rows[t] (int32; negative:
    padding, nothing is stored), which lies in page tables[rows[t], positions[t] // page_size] at place
    positions[t] % page_size. With `frequencies` the keys are rotated as `rotary` does, and so is `q` [tokens, q_heads, dim],
    which is returned (in `q_out`, which may be q itself, or a new tensor); values are stored as they are. A row, position or
    page number outside the tables or the pool stores nothing and makes `check_device_status` raise PageError. No two
    tokens of a call may have the same place. Nothing is recorded for gradients.
    """
    _tensors(k, v, k_pages, v_pages, tables, rows, positions)
    if k.dtype not in _STORAGE_OF or v.dtype != k.dtype or k_pages.dtype != k.dtype:
        raise ValueError('k, v and the pools must share dtype float32, float16 or bfloat16')
    k_token, k_head = _heads(k, 'k')
    v_token, v_head = (k_token, k_head) if v.stride() == k.stride() and v.shape == k.shape else _heads(v, 'v')
    pages, pool_heads, page_size, pool_dim, page_stride, page_head_stride, sequences, width, table_stride = _pools(k_pages, v_pages, tables)
    tokens, kv_heads, dim = k.shape
    if v.shape != k.shape or pool_heads != kv_heads or pool_dim != dim:
        raise ValueError('k, v and the pools disagree in shape')
    if (pages > 1 and page_stride == 0) or (kv_heads > 1 and page_head_stride == 0):
        raise ValueError('the pools must not be expanded tensors: they are written')
    _index(rows, 'rows', tokens)
    _index(positions, 'positions', tokens, wide=True)
    pairs = _rotation(frequencies, layout, dim)
    q_heads = q_token = q_head = q_out_token = q_out_head = 0
    if q is None and q_out is not None:
        raise ValueError('q_out without q')
    if q is not None:
        _tensors(q)
        q_token, q_head = _heads(q, 'q')
        q_heads = q.shape[1]
        if q.dtype != k.dtype or q.shape[0] != tokens or q.shape[2] != dim:
            raise ValueError('q must be a [tokens, q_heads, dim] tensor of the dtype of k')
        if q_out is not None:
            _tensors(q_out)
            if q_out.dtype != q.dtype or q_out.shape != q.shape:
                raise ValueError('q_out must have the shape and dtype of q')
            q_out_token, q_out_head = _heads(q_out, 'q_out', written=True)
            if q_out.data_ptr() == q.data_ptr() and (q_out_token, q_out_head) != (q_token, q_head):
                raise ValueError('q_out must be q itself or lie elsewhere')
    _on_current_device(k, v, k_pages, v_pages, tables, rows, positions, *[x for x in (frequencies, q, q_out) if x is not None])
    if q is not None and q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        q_out_token, q_out_head = q_heads * dim, dim
    native.call('dtn_paged_append', native.PAGED_APPEND_ARGS.pack(
        k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), tables.data_ptr(), rows.data_ptr(), positions.data_ptr(),
        frequencies.data_ptr() if pairs else 0, q.data_ptr() if q_heads else 0, q_out.data_ptr() if q_heads else 0,
        positions.dtype is torch.int64, tokens, kv_heads, dim, k_token, k_head, v_token, v_head, pages, page_size, page_stride,
        page_head_stride, sequences, width, table_stride, pairs, _LAYOUTS[layout], q_heads, q_token, q_head, q_out_token, q_out_head,
        _STORAGE_OF[k.dtype], float(amplitude)), _stream())
    return q_out


_paged_workspaces: dict[tuple[int, int], tuple[torch.Tensor, int, int]] = {}
_PAGED_COUNTER_BYTES = 4096


def _paged_workspace(q: torch.Tensor, stream: int) -> tuple[torch.Tensor, int, int]:
    """The parts and counters of `paged_attention`, its address and size: one workspace per device and stream (15 MB, kept as the
    products' are). Its counters are zeroed here once; every call leaves them zero. A call that is captured gets one of its own from
    the graph's memory, zeroed by each replay: replays may run beside one another and beside eager calls. The caller holds the
    tensor until its launch is queued; of threads that make a stream's first call at once all get the workspace of one."""
    capturing = torch.cuda.is_current_stream_capturing()
    key = (q.get_device(), stream)
    held = None if capturing else _paged_workspaces.get(key)
    if held is None:
        size = ct.c_size_t(0)
        native.call('dtn_paged_attention_workspace_bytes', ct.byref(size))
        workspace = torch.empty(size.value, dtype=torch.uint8, device=q.device)
        workspace[:_PAGED_COUNTER_BYTES].zero_()
        held = workspace, workspace.data_ptr(), size.value
        if not capturing:
            held = _paged_workspaces.setdefault(key, held)
    return held


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, scale: float,
                    rows: torch.Tensor | None = None, window: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over a paged key-value cache: q[n, q_heads, dim] -> out[n, q_heads, dim].

    Pools and tables as in `paged_append`; lengths: int32 [sequences], the tokens of each that are seen (the new one among
    them). rows: int32 [n], the sequence of each query (None: query i is sequence i); a negative row (padding of a captured
    batch) and a length of zero give zeros. window > 0 keeps the last `window` tokens only. Query head h reads kv head
    h // (q_heads // kv_heads). Heads have a multiple of 16 bytes (at most 256 elements) and start on 16-byte boundaries in the
    pools. Storage float32 / float16 / bfloat16, softmax and sums in FP32 (float16: a probability counts to 2^-23 of itself or 2^-44
    of the largest, whichever is more); `out` is float32 by default, as
    `gqa_attention` returns it, or a given tensor of float32 or of q's dtype, which may be q itself but must not overlap q or the
    pools otherwise. The values in a page behind a sequence's end do
    not matter, NaN included. A row or length outside the tables, or a page number outside the pool, makes
    `check_device_status` raise PageError; a sequence with such a page gets NaN. Nothing is recorded for gradients.
    """
    _tensors(q, k_pages, v_pages, tables, lengths)
    if q.dtype not in _STORAGE_OF or k_pages.dtype != q.dtype:
        raise ValueError('q and the pools must share dtype float32, float16 or bfloat16')
    q_token, q_head = _heads(q, 'q')
    pages, kv_heads, page_size, pool_dim, page_stride, page_head_stride, sequences, width, table_stride = _pools(k_pages, v_pages, tables)
    count, q_heads, dim = q.shape
    if pool_dim != dim:
        raise ValueError('q and the pools disagree in the head size')
    if kv_heads == 0 or q_heads % kv_heads:
        raise ValueError('query heads must be a multiple of kv heads')
    _index(lengths, 'lengths', sequences)
    if rows is not None:
        _tensors(rows)
        _index(rows, 'rows', count)
    elif count > sequences:
        raise ValueError(f'{count} queries but {sequences} sequences')
    if type(window) is not int or not 0 <= window < 1 << 63:
        raise ValueError(f'window must be a non-negative integer, got {window!r}')
    scale = float(scale)
    if out is not None:
        _tensors(out)
        if out.shape != q.shape or out.dtype not in (torch.float32, q.dtype):
            raise ValueError('out must have the shape of q and dtype float32 or that of q')
        out_token, out_head = _heads(out, 'out', written=True)
        if out.data_ptr() == q.data_ptr() and q.numel() and (out.dtype != q.dtype or (out_token, out_head) != (q_token, q_head)):
            raise ValueError('out must be q itself or lie elsewhere')
    _on_current_device(q, k_pages, v_pages, tables, lengths, *[x for x in (rows, out) if x is not None])
    if out is None:
        out = torch.empty_like(q, dtype=torch.float32, memory_format=torch.contiguous_format)
        out_token, out_head = q_heads * dim, dim
    stream = _stream()
    held, workspace, workspace_bytes = _paged_workspace(q, stream)
    native.call('dtn_paged_attention', native.PAGED_ATTENTION_ARGS.pack(
        q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), tables.data_ptr(), lengths.data_ptr(), 0 if rows is None else rows.data_ptr(),
        out.data_ptr(), workspace, workspace_bytes, count, q_heads, kv_heads, dim, q_token, q_head, out_token, out_head, pages, page_size,
        page_stride, page_head_stride, sequences, width, table_stride, window, _STORAGE_OF[q.dtype], out.dtype is torch.float32, scale), stream)
    return out


def copy_pages(pages: torch.Tensor, sources: torch.Tensor, destinations: torch.Tensor) -> None:
    """Copies page sources[i] onto page destinations[i] for every i, in one launch.

    pages: [pages, kv_heads, page_size, dim] with dense pages, or with one or two leading dimensions (layers; keys and
    values), in each of which the same pages are copied. sources, destinations: int32 [n]. No destination may occur twice or
    be a source. A page number outside the pool copies nothing and makes `check_device_status` raise PageError.
    """
    _tensors(pages, sources, destinations)
    shape = pages.shape
    if len(shape) == 5:
        planes, count, heads, size, dim = shape
    elif len(shape) == 4:
        planes, (count, heads, size, dim) = 1, shape
    elif len(shape) == 6:
        layers, kinds, count, heads, size, dim = shape
        planes = layers * kinds
    else:
        raise ValueError('pages must be a [pages, kv_heads, page_size, dim] tensor, or one with one or two leading dimensions')
    dense = heads * size * dim
    page_stride, plane_stride = dense, count * dense
    if not pages.is_contiguous():
        strides = pages.stride()
        for extent, stride, expected in zip(shape[-3:], strides[-3:], (size * dim, dim, 1)):
            if extent > 1 and stride != expected:
                raise ValueError('the values of one page must be dense')
        page_stride = strides[-4] if count > 1 else dense
        leading = [(extent, stride) for extent, stride in zip(shape[:-4], strides[:-4]) if extent > 1]
        plane_stride = leading[-1][1] if leading else 0
        if len(leading) == 2 and leading[0][1] != leading[1][0] * plane_stride:
            raise ValueError('the leading dimensions of pages must be evenly spaced')
        if dense and (page_stride < dense or (planes > 1 and plane_stride == 0)):
            raise ValueError('pages must not be an expanded tensor: it is written')
    _index(sources, 'sources')
    _index(destinations, 'destinations', sources.shape[0])
    _on_current_device(pages, sources, destinations)
    unit = pages.element_size()
    native.call('dtn_copy_pages', pages.data_ptr(), planes, plane_stride * unit, count, page_stride * unit, dense * unit, sources.data_ptr(),
                destinations.data_ptr(), sources.shape[0], _stream())


def check_device_status() -> None:
    """Synchronises the current stream and raises if a kernel reported a wait that ran out (DeviceWaitError) or a page number,
    position, row or length that a paged cache does not cover (PageError); the first report since the last check. An operator of a
    paged cache that is captured as the first call on a device reports nothing: call it once, or make a PagedCache, before."""
    native.raise_on_device_status(_stream())
