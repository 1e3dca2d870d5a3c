"""Host-side mirror of the reference's launch API (namespace mgt_cuda) over the C ABI.

Names follow the reference: RandomWalkKernelConfig / LaunchRandomWalkKernel
(native/cuda/mgt_cuda/random_walk_kernel.cuh), CudaMlpShape / MlpLossGradWorkspaceFloats /
LaunchMlpLossGrad... (native/cuda/mgt_cuda/mlp_backward.cuh), AdamWKernelConfig /
LaunchAdamWKernel[WithHalfMirror] (native/cuda/mgt_cuda/adamw.cuh). Functions return the
reference's status codes as ints; device buffers are torch CUDA tensors owned by the caller.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

from . import _lib

STATUS = {0: "ok", 1: "invalid_config", 2: "invalid_puzzle", 3: "capacity_exceeded", 4: "cuda_failure",
          5: "nccl_failure", 6: "io_failure", 7: "device_timeout"}


class MgtError(RuntimeError):
    def __init__(self, status: int, what: str):
        super().__init__(f"{what}: status {status} ({STATUS.get(status, 'unknown')})")
        self.status = status


def status_name(status: int) -> str:
    return _lib.load().mgt_status_name(status).decode()


def _ptr(t):
    if t is None:
        return None
    if hasattr(t, "data_ptr"):
        return C.c_void_p(t.data_ptr())
    return C.c_void_p(int(t))


def _stream(stream):
    if stream is None:
        import torch
        stream = torch.cuda.current_stream()
    return C.c_void_p(stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream))


# element types of the operators that take more than one (MGT_F32, MGT_F16, MGT_BF16)
F32, F16, BF16 = 0, 1, 2


_torch = None
_DTYPES = _CODES = _call = None


class _Unfit(Exception):
    """A tensor that cannot stand for what an argument asks for."""


def _with_torch():
    """torch and the library, loaded on first use."""
    global _torch, _DTYPES, _CODES, _call
    if _torch is None:
        import torch
        _DTYPES = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
        _CODES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}
        _call = _lib.load()
        _torch = torch
    return _torch


def _address(t, type_code, elements, device):
    """The address behind a dense tensor that holds `elements` of a type. Another type, another device than `device` (the host
    included), too few elements, or some that do not lie side by side, raise _Unfit; None and plain addresses are the library's to judge."""
    try:
        if t.dtype is not _DTYPES.get(type_code) or t.get_device() != device:
            raise _Unfit
    except AttributeError:  # no tensor
        return t
    if not t.is_contiguous() or t.numel() < elements:
        raise _Unfit
    return t.data_ptr()


def _rows_address(t, type_code, elements, device, rows):
    """The same for rows = (rows, columns, pitch), which may be a view too: of rows that lie so far apart."""
    try:
        if t.dtype is not _DTYPES.get(type_code) or t.get_device() != device:
            raise _Unfit
    except AttributeError:
        return t
    if t.is_contiguous():
        if t.numel() < elements:
            raise _Unfit
    elif not _lies_in_rows(t, *rows) or t.untyped_storage().nbytes() // t.element_size() - t.storage_offset() < elements:
        raise _Unfit
    return t.data_ptr()


def _lies_in_rows(t, rows, cols, pitch):
    """Whether a view's last dimension lies side by side and the ones before it, taken together, are `rows` rows `pitch` apart, or more."""
    dims = [(n, step) for n, step in zip(t.shape, t.stride()) if n != 1]
    if cols == 1 and dims[-1][1] != 1:  # (a column of a matrix)
        dims.append((1, 1))
    if dims[-1][1] != 1:
        return False
    have = 1
    for n, step in reversed(dims[:-1]):
        if step != pitch * have:
            return False
        have *= n
    return have >= rows


def _raw_stream(stream, device):
    """The cudaStream_t of a stream, of the current one where there is none (without building an object for it: 1.5 us)."""
    if stream is None:
        return _torch._C._cuda_getCurrentRawStream(device)
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _current_device(stream):
    """The current device, of which tensors have to be. With plain addresses and a stream nothing is asked of torch's CUDA side."""
    torch = _torch or _with_torch()
    return torch.cuda.current_device() if stream is None or torch.cuda.is_initialized() else None


class _WalkCfg(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in ("sample_count", "k_min", "k_max", "move_count", "state_len", "state_storage_len")]


class _Shape(C.Structure):
    _fields_ = [(n, C.c_uint32) for n in ("state_len", "state_value_pad", "hd1", "hd2", "residual_blocks", "output_dim")]


class _Adam(C.Structure):
    _fields_ = [("param_count", C.c_uint64), ("step", C.c_uint64), ("learning_rate", C.c_float), ("beta1", C.c_float),
                ("beta2", C.c_float), ("eps", C.c_float), ("weight_decay", C.c_float)]


class _LayerNorm(C.Structure):
    """mgt_layer_norm_config_t"""
    _fields_ = [("rows", C.c_uint32), ("cols", C.c_uint32), ("eps", C.c_float), ("x_type", C.c_int32), ("y_type", C.c_int32), ("dx_type", C.c_int32),
                ("x_pitch", C.c_uint64), ("y_pitch", C.c_uint64), ("dx_pitch", C.c_uint64)]


class _Tensor(C.Structure):
    """mgt_tensor_t"""
    _fields_ = [("data", C.c_void_p), ("count", C.c_uint64), ("type", C.c_int32), ("reserved", C.c_int32)]


class BackwardProfile(C.Structure):
    """mgt_cuda::MlpBackwardProfile (native/cuda/mgt_cuda/mlp_backward.cuh:11-19)."""
    _fields_ = [(n, C.c_float) for n in ("input_forward_ms", "hidden_forward_ms", "residual_forward_ms", "output_ms",
                                         "residual_backward_ms", "hidden_backward_ms", "input_grad_ms")]


@dataclass
class RandomWalkKernelConfig:
    sample_count: int = 0
    k_min: int = 0
    k_max: int = 0
    move_count: int = 18
    state_len: int = 72
    state_storage_len: int = 80

    def c(self):
        return _WalkCfg(self.sample_count, self.k_min, self.k_max, self.move_count, self.state_len, self.state_storage_len)


@dataclass
class CudaMlpShape:
    state_len: int
    state_value_pad: int
    hd1: int
    hd2: int
    residual_blocks: int
    output_dim: int = 1

    def c(self):
        return _Shape(self.state_len, self.state_value_pad, self.hd1, self.hd2, self.residual_blocks, self.output_dim)

    @property
    def param_count(self) -> int:
        shape = self.c()
        return int(_lib.load().mgt_mlp_param_count(C.byref(shape)))


@dataclass
class AdamWKernelConfig:
    param_count: int
    step: int
    learning_rate: float
    beta1: float = 0.9
    beta2: float = 0.999
    eps: float = 1e-8
    weight_decay: float = 0.0

    def c(self):
        return _Adam(self.param_count, self.step, self.learning_rate, self.beta1, self.beta2, self.eps, self.weight_decay)


def launch_expand_scalar_labels(scalar_labels, sample_count: int, output_dim: int, expanded_labels, stream=None) -> int:
    """ExpandScalarLabelsKernel (native/tools/mgt_native_train_smoke.cu:74-80): labels[b][o] = scalar[b] for every output."""
    return int(_lib.load().mgt_launch_expand_scalar_labels(_ptr(scalar_labels), sample_count, output_dim, _ptr(expanded_labels), _stream(stream)))


def validate_random_walk_kernel_config(config: RandomWalkKernelConfig) -> int:
    cfg = config.c()
    return int(_lib.load().mgt_validate_random_walk_config(C.byref(cfg)))


def launch_random_walk_kernel(config, base_seed, epoch, step, global_rank, device_moves, device_target, device_states,
                              device_labels, device_meta, stream=None) -> int:
    cfg = config.c()
    return int(_lib.load().mgt_launch_random_walk(C.byref(cfg), base_seed & (2**64 - 1), epoch, step, global_rank,
                                                  _ptr(device_moves), _ptr(device_target), _ptr(device_states),
                                                  _ptr(device_labels), _ptr(device_meta), _stream(stream)))


def load_puzzle_definition(group_json: str, target_bin: str, group_id: int = 888, state_len: int = 72, move_count: int = 18):
    """LoadPuzzleDefinition (native/src/puzzle_io.cpp:48-97): returns (status, moves[18][80] uint8, target[80] uint8)."""
    import numpy as np
    moves = np.zeros((18, 80), np.uint8)
    target = np.zeros(80, np.uint8)
    lib = _lib.load()
    lib.mgt_load_puzzle_definition.argtypes = [C.c_char_p, C.c_char_p, C.c_uint32, C.c_uint32, C.c_uint32, C.c_void_p, C.c_void_p]
    st = int(lib.mgt_load_puzzle_definition(str(group_json).encode(), str(target_bin).encode(), group_id, state_len, move_count,
                                            moves.ctypes.data_as(C.c_void_p), target.ctypes.data_as(C.c_void_p)))
    return st, moves, target


def validate_cuda_mlp_shape(shape: CudaMlpShape) -> int:
    s = shape.c()
    return int(_lib.load().mgt_validate_mlp_shape(C.byref(s)))


class _TrainOptions(C.Structure):
    """mgt_train_options_t"""
    _fields_ = [("operand_format", C.c_int32), ("loss_kind", C.c_int32), ("batch_norm", C.c_int32), ("bn_eps", C.c_float)]


def mlp_loss_grad_workspace_floats(shape, sample_count, input_grad_partial_chunks=1, use_half_input_grad=True,
                                   use_half_linear=True, batch_norm=False, layer_norm=False) -> int:
    s = shape.c()
    lib = _lib.load()
    if layer_norm:  # (neither beside batch normalisation nor all in fp32)
        return 0 if batch_norm or not use_half_linear else lib.mgt_mlp_loss_grad_workspace_floats_with_layer_norm(
            C.byref(s), sample_count, input_grad_partial_chunks, int(use_half_input_grad))
    if not batch_norm:
        return int(lib.mgt_mlp_loss_grad_workspace_floats(C.byref(s), sample_count, input_grad_partial_chunks,
                                                          int(use_half_input_grad), int(use_half_linear)))
    opt = _TrainOptions(0, 0, 1, 1e-5)
    lib.mgt_mlp_loss_grad_workspace_floats_with_options.restype = C.c_uint64
    lib.mgt_mlp_loss_grad_workspace_floats_with_options.argtypes = [C.c_void_p, C.c_uint32, C.c_uint32, C.c_int32, C.c_int32, C.c_void_p]
    return int(lib.mgt_mlp_loss_grad_workspace_floats_with_options(C.byref(s), sample_count, input_grad_partial_chunks,
                                                                   int(use_half_input_grad), int(use_half_linear), C.byref(opt)))


def bn_param_count(shape) -> int:
    """mgt_bn_param_count: floats of batch-norm scale/shift that follow the reference's parameters (2 * (blocks + 1) * hd2)."""
    s = shape.c()
    lib = _lib.load()
    lib.mgt_bn_param_count.restype = C.c_uint64
    lib.mgt_bn_param_count.argtypes = [C.c_void_p]
    return int(lib.mgt_bn_param_count(C.byref(s)))


def fold_batch_norm(shape, weights, scale_shift, running_stats, eps: float = 1e-5):
    """mgt_fold_batch_norm on host arrays: a copy of `weights` (the reference's layout) with the normalisation folded into
    the hidden layer and into every block's fc2, using the running statistics. Raises MgtError on a bad argument."""
    import numpy as np
    s = shape.c()
    lib = _lib.load()
    out = np.array(weights, dtype=np.float32, copy=True).ravel()
    ss = np.ascontiguousarray(scale_shift, dtype=np.float32).ravel()
    rs = np.ascontiguousarray(running_stats, dtype=np.float32).ravel()
    n = bn_param_count(shape)
    if out.size != shape.param_count or ss.size != n or rs.size != n:
        raise MgtError(1, "fold_batch_norm: array sizes")
    lib.mgt_fold_batch_norm.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_float]
    st = int(lib.mgt_fold_batch_norm(C.byref(s), out.ctypes.data_as(C.c_void_p), ss.ctypes.data_as(C.c_void_p), rs.ctypes.data_as(C.c_void_p), eps))
    if st != 0:
        raise MgtError(st, "fold_batch_norm")
    return out


STATS_EXCHANGE_FN = C.CFUNCTYPE(C.c_int32, C.c_void_p, C.c_void_p, C.c_uint64, C.c_void_p)
GRADIENT_READY_FN = C.CFUNCTYPE(C.c_int32, C.c_void_p, C.c_uint32, C.c_uint64, C.c_uint64, C.c_void_p)


class Engine:
    """Owner of the opaque engine handle (stands where the reference passes cuBLAS handles)."""

    def __init__(self, device_id: int = 0):
        self._lib = _lib.load()
        handle = C.c_void_p()
        st = self._lib.mgt_engine_create(device_id, C.byref(handle))
        if st != 0:
            raise MgtError(st, "mgt_engine_create")
        self.handle = handle

    def close(self):
        if getattr(self, "handle", None):
            self._lib.mgt_engine_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def launch_count(self) -> int:
        return int(self._lib.mgt_engine_launch_count(self.handle))

    @property
    def fork_count(self) -> int:
        return int(self._lib.mgt_engine_fork_count(self.handle))

    def check(self, stream=None):
        code = C.c_int32(0)
        st = int(self._lib.mgt_engine_check(self.handle, _stream(stream), C.byref(code)))
        return st, int(code.value)

    def set_train_options(self, bf16: bool = False, cross_entropy: bool = False, batch_norm: bool = False, bn_eps: float = 1e-5) -> int:
        """mgt_engine_set_train_options: bfloat16 operands, cross-entropy on depth - 1, batch normalisation (defaults = the reference)."""
        opt = _TrainOptions(int(bf16), int(cross_entropy), int(batch_norm), float(bn_eps))
        self._lib.mgt_engine_set_train_options.argtypes = [C.c_void_p, C.c_void_p]
        return int(self._lib.mgt_engine_set_train_options(self.handle, C.byref(opt)))

    def set_batch_norm_state(self, running_stats=None, momentum: float = 0.1, world_size: int = 1, exchange_buffer=None, exchange=None) -> int:
        """mgt_engine_set_batch_norm_state. `exchange(user, device_pointer, float_count, stream) -> status` must enqueue an
        in-place average of the buffer over all ranks on `stream`; `exchange_buffer` is a device tensor or a raw pointer."""
        cb = STATS_EXCHANGE_FN(exchange) if exchange is not None else None
        self._stats_keepalive = (cb, running_stats, exchange_buffer)
        buf = exchange_buffer if isinstance(exchange_buffer, int) or exchange_buffer is None else _ptr(exchange_buffer)
        self._lib.mgt_engine_set_batch_norm_state.argtypes = [C.c_void_p, C.c_void_p, C.c_float, C.c_uint32, C.c_void_p, C.c_void_p, C.c_void_p]
        return int(self._lib.mgt_engine_set_batch_norm_state(self.handle, _ptr(running_stats), momentum, world_size, buf,
                                                             C.cast(cb, C.c_void_p) if cb is not None else None, None))

    def set_layer_norm(self, enabled: bool = True, eps: float = 1e-5) -> int:
        """mgt_engine_set_layer_norm: layer normalisation where batch normalisation would be, every sample by itself."""
        return self._lib.mgt_engine_set_layer_norm(self.handle, int(enabled), eps)

    def set_early_range_hook(self, fn=None) -> int:
        """mgt_engine_set_early_range_hook: fn(user, ready_id, offset, count, stream) -> status, or None to remove it."""
        cb = GRADIENT_READY_FN(fn) if fn is not None else None
        self._early_keepalive = cb
        self._lib.mgt_engine_set_early_range_hook.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
        return int(self._lib.mgt_engine_set_early_range_hook(self.handle, C.cast(cb, C.c_void_p) if cb is not None else None, None))

    def launch_mlp_loss_grad(self, shape, device_weights, device_weights_half, device_states, device_labels, sample_count,
                             device_loss, device_grad, workspace, workspace_floats, input_grad_partial_chunks=1,
                             input_grad_positions_per_block=1, use_half_input_grad=True, use_half_linear=True,
                             profile=None, gradient_ready=None, stream=None, input_grad_position_tile=0) -> int:
        """LaunchMlpLossGrad...ExternalHalf (native/cuda/mgt_cuda/mlp_backward.cuh:224-287)."""
        s = shape.c()
        cb = GRADIENT_READY_FN(gradient_ready) if gradient_ready is not None else None
        self._keepalive = cb
        return int(self._lib.mgt_launch_mlp_loss_grad(
            self.handle, C.byref(s), _ptr(device_weights), _ptr(device_weights_half), _ptr(device_states), _ptr(device_labels),
            sample_count, _ptr(device_loss), _ptr(device_grad), _ptr(workspace), workspace_floats, input_grad_partial_chunks,
            input_grad_positions_per_block, int(use_half_input_grad), int(use_half_linear),
            C.byref(profile) if profile is not None else None, C.cast(cb, C.c_void_p) if cb is not None else None, None,
            _stream(stream), input_grad_position_tile))

    def debug_gemm(self, a, lda, a_mn_major, b, ldb, b_mn_major, d, m, n, k, splits=1, partial=None, stream=None) -> int:
        return int(self._lib.mgt_debug_gemm(self.handle, _ptr(a), lda, int(a_mn_major), _ptr(b), ldb, int(b_mn_major), _ptr(d),
                                            m, n, k, splits, _ptr(partial), _stream(stream)))

    def debug_sums(self, src, terms, items, jobs, planes, dst, stream=None) -> int:
        return int(self._lib.mgt_debug_sums(self.handle, _ptr(src), terms, items, jobs, int(planes), _ptr(dst), _stream(stream)))


def validate_adamw_kernel_config(config: AdamWKernelConfig) -> int:
    cfg = config.c()
    return int(_lib.load().mgt_validate_adamw_config(C.byref(cfg)))


def launch_adamw_kernel(config, device_weights, device_grad, device_m, device_v, stream=None) -> int:
    cfg = config.c()
    return int(_lib.load().mgt_launch_adamw(C.byref(cfg), _ptr(device_weights), _ptr(device_grad), _ptr(device_m),
                                            _ptr(device_v), _stream(stream)))


def launch_adamw_kernel_with_half_mirror(config, device_weights, device_weights_half, device_grad, device_m, device_v,
                                         stream=None) -> int:
    cfg = config.c()
    return int(_lib.load().mgt_launch_adamw_with_half_mirror(C.byref(cfg), _ptr(device_weights), _ptr(device_weights_half),
                                                             _ptr(device_grad), _ptr(device_m), _ptr(device_v), _stream(stream)))


def launch_float_to_half(device_values, count, device_half, stream=None) -> int:
    return int(_lib.load().mgt_launch_float_to_half(_ptr(device_values), count, _ptr(device_half), _stream(stream)))


def launch_adamw_kernel_with_clip(config, device_weights, device_weights_half, device_grad, device_clip, device_m, device_v, stream=None) -> int:
    """mgt_launch_adamw_with_clip: the update of a gradient scaled by device_clip[1], skipped where the norm device_clip[0] is not finite
    (what launch_gradient_norm leaves). device_weights_half may be None. A tensor of another type, on another device than the
    current one, too small, or not dense, is refused (1)."""
    n, d = config.param_count, _current_device(stream)
    try:
        w, half = _address(device_weights, F32, n, d), _address(device_weights_half, F16, n, d)
        grad, clip, m, v = _address(device_grad, F32, n, d), _address(device_clip, F32, 2, d), _address(device_m, F32, n, d), _address(device_v, F32, n, d)
    except _Unfit:
        return 1
    return _call.mgt_launch_adamw_with_clip(C.byref(config.c()), w, half, grad, clip, m, v, _raw_stream(stream, d))


@dataclass(frozen=True)
class LayerNormConfig:
    """mgt_layer_norm_config_t. y_type and y_pitch are those of dy in the backward pass; dx_type None = x_type; a pitch of 0 = cols."""
    rows: int
    cols: int
    eps: float = 1e-5
    x_type: int = F32
    y_type: int = F32
    dx_type: int | None = None
    x_pitch: int = 0
    y_pitch: int = 0
    dx_pitch: int = 0

    def __post_init__(self):
        fits = 0 <= self.rows < 2**32 and 0 <= self.cols < 2**32 and min(self.x_pitch, self.y_pitch, self.dx_pitch) >= 0
        dx_type = self.x_type if self.dx_type is None else self.dx_type
        # (what a field would wrap around is refused as a config without columns)
        c = _LayerNorm(self.rows, self.cols, self.eps, self.x_type, self.y_type, dx_type, self.x_pitch, self.y_pitch, self.dx_pitch) if fits else _LayerNorm()
        pitches = [pitch or self.cols for pitch in (self.x_pitch, self.y_pitch, self.dx_pitch)]
        extents = tuple((self.rows - 1) * pitch + self.cols if self.rows else 0 for pitch in pitches)
        layouts = tuple((self.rows, self.cols, pitch) for pitch in pitches)
        for name, value in (("_c", c), ("_reference", C.byref(c)), ("_extents", extents + layouts), ("_dx_type", dx_type)):
            object.__setattr__(self, name, value)

    def c(self):
        return self._c


def validate_layer_norm_config(config: LayerNormConfig) -> int:
    return _lib.load().mgt_validate_layer_norm_config(config._reference)


def launch_layer_norm(config: LayerNormConfig, x, gamma, beta, y, mean=None, rstd=None, stream=None) -> int:
    """mgt_launch_layer_norm: y = gamma * (x - mean) * rstd + beta over the columns of every row; gamma, beta, mean and rstd may be None.
    A tensor of another type, on another device than the current one, or too small, is refused (1), and so are one that is not dense and, for x
    and y, a view whose rows do not lie as the config says."""
    d = _current_device(stream)
    x_extent, y_extent, _, x_rows, y_rows, _ = config._extents
    rows, cols = config.rows, config.cols
    try:
        x, y = _rows_address(x, config.x_type, x_extent, d, x_rows), _rows_address(y, config.y_type, y_extent, d, y_rows)
        gamma, beta, mean, rstd = _address(gamma, F32, cols, d), _address(beta, F32, cols, d), _address(mean, F32, rows, d), _address(rstd, F32, rows, d)
    except _Unfit:
        return 1
    return _call.mgt_launch_layer_norm(config._reference, x, gamma, beta, y, mean, rstd, _raw_stream(stream, d))


def layer_norm_backward_workspace_floats(config: LayerNormConfig) -> int:
    return _lib.load().mgt_layer_norm_backward_workspace_floats(config._reference)


def launch_layer_norm_backward(config: LayerNormConfig, dy, x, gamma, mean, rstd, dx, dgamma, dbeta, dbias, workspace, workspace_floats, stream=None) -> int:
    """mgt_launch_layer_norm_backward: dx, and the sums over the rows dgamma, dbeta and dbias (each may be None). Tensors as above."""
    d = _current_device(stream)
    x_extent, dy_extent, dx_extent, x_rows, dy_rows, dx_rows = config._extents
    rows, cols = config.rows, config.cols
    try:
        dy, x = _rows_address(dy, config.y_type, dy_extent, d, dy_rows), _rows_address(x, config.x_type, x_extent, d, x_rows)
        dx = _rows_address(dx, config._dx_type, dx_extent, d, dx_rows)
        gamma, mean, rstd = _address(gamma, F32, cols, d), _address(mean, F32, rows, d), _address(rstd, F32, rows, d)
        dgamma, dbeta, dbias = _address(dgamma, F32, cols, d), _address(dbeta, F32, cols, d), _address(dbias, F32, cols, d)
        workspace = _address(workspace, F32, workspace_floats, d)
    except _Unfit:
        return 1
    return _call.mgt_launch_layer_norm_backward(config._reference, dy, x, gamma, mean, rstd, dx, dgamma, dbeta, dbias, workspace, workspace_floats,
                                                _raw_stream(stream, d))


class TensorList:
    """An array of mgt_tensor_t for the gradient-norm calls, and the tensors it stands for: float32, float16 or bfloat16, each dense,
    all on one CUDA device. Built once where gradients stay in place: it stands for the memory that they have then, and holds that, whatever
    becomes of a tensor (another `.data`, say) later. Not for memory that is taken away behind it (`untyped_storage().resize_`)."""

    def __init__(self, tensors):
        _with_torch()
        self.tensors = list(tensors)
        self.count = len(self.tensors)
        self._array = (_Tensor * max(1, self.count))()
        devices = set()
        for entry, t in zip(self._array, self.tensors):
            kind = _CODES.get(t.dtype)
            if kind is None or not t.is_contiguous() or not t.is_cuda:
                raise MgtError(1, "TensorList: dense CUDA tensors of float32, float16 or bfloat16")
            entry.data, entry.count, entry.type = t.data_ptr(), t.numel(), kind
            devices.add(t.get_device())
        if len(devices) != 1:
            raise MgtError(1, "TensorList: tensors of one device")
        self._memory = [t.untyped_storage() for t in self.tensors]
        self.device = devices.pop()
        self.pointer = C.addressof(self._array)


def gradient_norm_workspace_floats(tensors: TensorList) -> int:
    return _call.mgt_gradient_norm_workspace_floats(tensors.pointer, tensors.count)


def launch_gradient_norm(tensors: TensorList, max_norm: float, result, tensor_norms, workspace, workspace_floats, stream=None) -> int:
    """mgt_launch_gradient_norm: result = {norm over all tensors, scale that brings it to max_norm at most}; tensor_norms (may be None) = the norm of each."""
    d = _current_device(stream)
    if tensors.device != d:
        return 1
    try:
        result, norms, workspace = _address(result, F32, 2, d), _address(tensor_norms, F32, tensors.count, d), _address(workspace, F32, workspace_floats, d)
    except _Unfit:
        return 1
    return _call.mgt_launch_gradient_norm(tensors.pointer, tensors.count, max_norm, result, norms, workspace, workspace_floats, _raw_stream(stream, d))


def launch_clip_gradients(tensors: TensorList, result, out_tensors: TensorList | None = None, stream=None) -> int:
    """mgt_launch_clip_gradients: every element times result[1], in place or into out_tensors (same counts and types). What is written
    overlaps neither another tensor of either list nor result (status 1)."""
    d = _current_device(stream)
    if tensors.device != d or (out_tensors is not None and (out_tensors.device != d or out_tensors.count != tensors.count)):
        return 1
    try:
        result = _address(result, F32, 2, d)
    except _Unfit:
        return 1
    return _call.mgt_launch_clip_gradients(tensors.pointer, tensors.count, result, out_tensors.pointer if out_tensors is not None else None, _raw_stream(stream, d))
