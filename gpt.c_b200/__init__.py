"""B200-native causal self-attention for gpt.c: ctypes access to ``libattn_sm100.so``.

The product is the C-ABI library declared in ``include/attn_sm100.h`` (hand-written sm_100a CUDA).
This package only loads it and offers a thin convenience layer that takes ``torch`` CUDA tensors
for device memory and streams; every call goes through the C ABI with raw pointers, the tensor-level
ones by way of a small extension module (``csrc/torch_calls.cpp``).  There is no
CPU or PyTorch fallback: if the library is missing or the device is not an sm_100 GPU the calls
raise.

The directory name contains a dot, so it cannot be imported with a plain ``import`` statement;
load it with ``importlib`` (see ``load_package`` in ``__graft_entry__.py``) under the module name
``gptc_b200``.
"""
from __future__ import annotations

import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "lib", "libattn_sm100.so")
CALLS_PATH = os.path.join(HERE, "lib", "gptc_b200_calls.so")
HEADER_PATH = os.path.join(HERE, "..", "include", "attn_sm100.h")

FLAG_FORCE_GENERIC = 1
FLAG_PREPARE_ONLY = 2
FLAG_CORE_ONLY = 4

# name -> (restype, argtypes); must list every function include/attn_sm100.h declares
_c = ctypes
SIGNATURES = {
    "attn_sm100_version": (_c.c_int, []),
    "attn_sm100_init": (_c.c_int, []),
    "attn_sm100_saved_bytes": (_c.c_size_t, [_c.c_int] * 4),
    "attn_sm100_backward_scratch_bytes": (_c.c_size_t, [_c.c_int] * 4),
    "attn_sm100_forward": (_c.c_int, [_c.c_void_p] * 5 + [_c.c_int] * 5 + [_c.c_void_p]),
    "attn_sm100_backward": (_c.c_int, [_c.c_void_p] * 6 + [_c.c_int] * 5 + [_c.c_void_p]),
    "attn_sm100_forward_static": (_c.c_int, [_c.c_void_p] * 3 + [_c.c_int] * 4 + [_c.c_void_p]),
    "attn_sm100_static_status": (_c.c_int, [_c.POINTER(_c.c_int), _c.c_int]),
    "attn_sm100_selftest_wait_limit": (_c.c_int, [_c.c_uint, _c.c_void_p]),
    "attn_sm100_paged_append": (_c.c_int, [_c.c_void_p] * 8 + [_c.c_longlong] * 2 + [_c.c_int] * 12 + [_c.c_void_p]),
    "attn_sm100_paged_forward": (_c.c_int, [_c.c_void_p] * 7 + [_c.c_longlong] * 2 + [_c.c_int] * 10 + [_c.c_float, _c.c_void_p]),
    "attn_sm100_device_status": (_c.c_int, [_c.POINTER(_c.c_int), _c.c_int]),
    "attn_sm100_strerror": (_c.c_char_p, [_c.c_int]),
    "linear_sm100_forward": (_c.c_int, [_c.c_void_p] * 5 + [_c.c_int] * 3 + [_c.c_void_p]),
    "linear_sm100_backward_scratch_bytes": (_c.c_size_t, [_c.c_int] * 3),
    "linear_sm100_backward": (_c.c_int, [_c.c_void_p] * 7 + [_c.c_int] * 3 + [_c.c_void_p]),
    "linear_sm100_backward_plan": (_c.c_int, [_c.c_int] * 6 + [_c.POINTER(_c.c_int)]),
    "layernorm_sm100_forward": (_c.c_int, [_c.c_void_p] * 3 + [_c.c_float] + [_c.c_void_p] * 3 + [_c.c_int] * 2 + [_c.c_void_p]),
    "layernorm_sm100_backward": (_c.c_int, [_c.c_void_p] * 8 + [_c.c_int] * 2 + [_c.c_void_p]),
    "tensor_sm100_fill": (_c.c_int, [_c.c_void_p, _c.c_size_t, _c.c_float, _c.c_void_p]),
    "tensor_sm100_arange": (_c.c_int, [_c.c_void_p, _c.c_size_t, _c.c_int, _c.c_int, _c.c_void_p]),
    "tensor_sm100_copy": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_size_t, _c.c_void_p]),
    "tensor_sm100_axpy": (_c.c_int, [_c.c_size_t, _c.c_float, _c.c_void_p, _c.c_void_p, _c.c_void_p]),
    "tensor_sm100_gelu_forward": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_size_t, _c.c_void_p]),
    "tensor_sm100_gelu_backward": (_c.c_int, [_c.c_void_p, _c.c_void_p, _c.c_void_p, _c.c_size_t, _c.c_void_p]),
    "tensor_sm100_embedding_forward": (_c.c_int, [_c.c_void_p] * 5 + [_c.c_longlong] * 3 + [_c.c_float] + [_c.c_int] * 6 + [_c.c_void_p]),
    "tensor_sm100_embedding_backward_scratch_bytes": (_c.c_size_t, [_c.c_longlong] + [_c.c_int] * 3),
    "tensor_sm100_embedding_backward": (_c.c_int, [_c.c_void_p] * 6 + [_c.c_longlong] * 4 + [_c.c_float] + [_c.c_int] * 7 + [_c.c_void_p]),
    "xent_sm100_forward": (_c.c_int, [_c.c_void_p] * 4 + [_c.c_int] * 2 + [_c.c_void_p]),
    "xent_sm100_selftest_wait_limit": (_c.c_int, [_c.c_void_p] * 4 + [_c.c_int] * 3 + [_c.c_uint, _c.c_void_p]),
    "xent_sm100_sample": (_c.c_int, [_c.c_void_p] * 7 + [_c.c_longlong] + [_c.c_int] * 2 + [_c.c_void_p]),
    "xent_sm100_linear_forward_scratch_bytes": (_c.c_size_t, [_c.c_void_p] * 2 + [_c.c_longlong] * 2 + [_c.c_int] * 4),
    "xent_sm100_linear_forward": (_c.c_int, [_c.c_void_p] * 6 + [_c.c_longlong] * 2 + [_c.c_int] * 5 + [_c.c_void_p]),
    "xent_sm100_selftest_linear_wait_limit": (_c.c_int, [_c.c_void_p] * 6 + [_c.c_longlong] * 2 + [_c.c_int] * 6 + [_c.c_void_p]),
    "xent_sm100_linear_backward_scratch_bytes": (_c.c_size_t, [_c.c_void_p] * 2 + [_c.c_longlong] * 2 + [_c.c_int] * 4),
    "xent_sm100_linear_backward": (_c.c_int, [_c.c_void_p] * 8 + [_c.c_longlong] * 3 + [_c.c_int] * 6 + [_c.c_void_p]),
    "xent_sm100_backward": (_c.c_int, [_c.c_void_p] * 4 + [_c.c_int] * 2 + [_c.c_void_p]),
    "adamw_sm100_step": (_c.c_int, [_c.c_void_p] * 5 + [_c.c_int] + [_c.c_float] * 5 + [_c.c_int, _c.c_void_p]),
}

_lib = None
_calls_module = None
_entry_classes = {}  # name of an entry point -> the class of its function in lib()


class AttnError(RuntimeError):
    def __init__(self, code: int, where: str):
        self.code = code
        msg = lib().attn_sm100_strerror(code).decode()
        super().__init__(f"{where} failed with status {code}: {msg}")


def lib() -> ctypes.CDLL:
    """Load libattn_sm100.so (once).  Raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(
                f"{LIB_PATH} is missing: build it with `python gpt.c_b200/build.py`; there is no fallback path")
        handle = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
            _entry_classes[name] = fn.__class__ = _entry_class(handle._FuncPtr)
        _lib = handle
        _shorten_calls()
    return _lib


def _entry_class(plain):
    """A class for one function of the library: a ctypes function like any other, which the extension module may give a
    shorter way from a call's arguments to the C ABI.  That way knows the signature above, so a function that is given
    another one becomes an ordinary ctypes function."""

    class Entry(plain):
        _flags_ = plain._flags_
        _restype_ = plain._restype_

        def __setattr__(self, name, value):
            if name in ("restype", "argtypes", "errcheck"):
                self.__class__ = plain
            plain.__setattr__(self, name, value)

        def __delattr__(self, name):
            if name in ("restype", "argtypes", "errcheck"):
                self.__class__ = plain
            plain.__delattr__(self, name)

    return Entry


def _shorten_calls():
    if _calls_module is not None:
        _calls_module.shorten_calls(_entry_classes)


def _calls():
    """The extension module over the C ABI (once).  Raises if it has not been built."""
    global _calls_module
    if _calls_module is None:
        import importlib.util

        import torch  # noqa: F401  (its libraries have to be loaded first)

        lib()
        if not os.path.exists(CALLS_PATH):
            raise FileNotFoundError(
                f"{CALLS_PATH} is missing: build it with `python gpt.c_b200/build.py`; there is no fallback path")
        spec = importlib.util.spec_from_file_location("gptc_b200_calls", CALLS_PATH)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        mod.set_error(AttnError)
        _calls_module = mod
        _shorten_calls()
    return _calls_module


def _raw(stream):
    return None if stream is None else stream.cuda_stream


def _check(code: int, where: str) -> None:
    if code != 0:
        raise AttnError(code, where)


def init() -> None:
    _check(lib().attn_sm100_init(), "attn_sm100_init")


def device_status(clear: bool = True) -> int:
    """Synchronise the current device and return its kernel status word (0 = fine)."""
    st = ctypes.c_int(0)
    rc = lib().attn_sm100_device_status(ctypes.byref(st), 1 if clear else 0)
    if rc not in (0, -6):
        raise AttnError(rc, "attn_sm100_device_status")
    return st.value


def static_status(clear: bool = True) -> int:
    """The same for the status word of attn_sm100_forward_static (a separate word inside the library)."""
    st = ctypes.c_int(0)
    rc = lib().attn_sm100_static_status(ctypes.byref(st), 1 if clear else 0)
    if rc not in (0, -6):
        raise AttnError(rc, "attn_sm100_static_status")
    return st.value


def saved_bytes(B: int, T: int, H: int, D: int) -> int:
    return lib().attn_sm100_saved_bytes(B, T, H, D)


def backward_scratch_bytes(B: int, T: int, H: int, D: int) -> int:
    return lib().attn_sm100_backward_scratch_bytes(B, T, H, D)


class Saved:
    """What forward leaves behind for backward (all device buffers, owned by torch)."""

    def __init__(self, saved, out, lse, shape, flags):
        self.saved, self.out, self.lse, self.shape, self.flags = saved, out, lse, shape, flags


def forward_into(qkv, out, out_copy, lse, saved, n_heads: int, flags: int = 0, stream=None) -> None:
    """Raw call: every buffer is supplied by the caller (torch CUDA tensors or None)."""
    _calls().forward_into(qkv, out, out_copy, lse, saved, n_heads, flags, _raw(stream))


def backward_into(saved, out, lse, dout, dqkv, scratch, n_heads: int, flags: int = 0, stream=None) -> None:
    _calls().backward_into(saved, out, lse, dout, dqkv, scratch, n_heads, flags, _raw(stream))


def forward(qkv, n_heads: int, flags: int = 0, keep_copy: bool = False):
    """qkv [B, T, 3C] fp32 CUDA tensor -> (out [B, T, C], Saved)."""
    out, out_copy, lse, saved, shape = _calls().forward(qkv, n_heads, flags, keep_copy)
    return out, Saved(saved, out if out_copy is None else out_copy, lse, shape, flags)


def backward(ctx: Saved, dout):
    """dout [B, T, C] -> dqkv [B, T, 3C] = [dq | dk | dv]."""
    return _calls().backward(ctx.saved, ctx.out, ctx.lse, dout, ctx.shape, ctx.flags)


# ---------------------------------------------------------------------------------------------
# Linear either side of the attention layer (include/linear_sm100.h); mirrors the reference's
# linear_forward_cuda_kernel / linear_backward_cuda_kernel (kernels/src/cuda/Linear.cu:37-92).
# ---------------------------------------------------------------------------------------------
def linear_forward(x, w, bias=None, planes=None, stream=None):
    """y[..., N] = x[..., K] @ w[N, K].T + bias.  `planes`: optional uint8 CUDA tensor of
    saved_bytes(...) bytes that receives y as bf16 hi/lo planes for the attention kernels."""
    return _calls().linear_forward(x, w, bias, planes, _raw(stream))


def linear_backward(dy, x, w, dw, db=None, stream=None, want_dx=True):
    """Returns dx = dy @ w (None when want_dx is false); accumulates dy.T @ x into dw (skipped when dw is
    None) and the column sums of dy into db."""
    return _calls().linear_backward(dy, x, w, dw, db, _raw(stream), want_dx)


# ---------------------------------------------------------------------------------------------
# LayerNorm (include/layernorm_sm100.h); mirrors layer_norm_{forward,backward}_cuda_kernel
# (kernels/src/cuda/LayerNorm.cu:115-165).
# ---------------------------------------------------------------------------------------------
def layernorm_forward(x, w, b=None, eps: float = 1e-5, stream=None):
    """Returns (y, mean, rstd) for x [..., C]."""
    return _calls().layernorm_forward(x, w, b, eps, _raw(stream))


def layernorm_backward(dy, x, mean, rstd, w, dw, db, dx, stream=None) -> None:
    """Accumulates into dw, db (may be None) and dx, like the reference."""
    _calls().layernorm_backward(dy, x, mean, rstd, w, dw, db, dx, _raw(stream))


# ---------------------------------------------------------------------------------------------
# Token and position embedding (include/tensor_sm100.h); the reference's is embedding_{forward,backward}_cuda_kernel
# (kernels/src/cuda/Embedding.cu:46-74).  Tables are fp32 or bf16 [rows, features], their rows may lie apart; tokens and positions are
# int32, int64, or fp32 as gpt.c has them.  One outside its table brings zeros, and no gradient.
# ---------------------------------------------------------------------------------------------
def embedding_forward(tokens, table, positions=None, pos_table=None, scale: float = 1.0, stream=None):
    """y[..., :] = scale * table[tokens] + pos_table[positions], of the type of the tables.  Without positions, a token's position is
    its index along the last dimension of tokens [..., T]; without pos_table nothing is added."""
    return _calls().embedding_forward(tokens, table, positions, pos_table, scale, _raw(stream))


def embedding_backward(dy, tokens, dtable, positions=None, dpos_table=None, scale: float = 1.0, stream=None) -> None:
    """Adds the gradients to dtable and dpos_table (either may be None), fp32 or bf16 whatever dy is: sums in fp32 and a fixed
    order, one rounding."""
    _calls().embedding_backward(dy, tokens, dtable, positions, dpos_table, scale, _raw(stream))


# ---------------------------------------------------------------------------------------------
# The vocabulary projection and its loss in one (include/xent_sm100.h): the logits, which the reference keeps three times over
# (src/transformer.c:107-108, kernels/src/cuda/CrossEntropyLoss.cu:8-129), are not in memory.  x and w are both fp32 or both bf16; x is
# contiguous or [rows, features] with rows apart, w and dw may have rows apart.  The calls do not record themselves for autograd.
# ---------------------------------------------------------------------------------------------
def linear_xent_forward(x, w, targets, stream=None):
    """Returns (losses, lse), fp32 of the shape of targets: the cross-entropy of each row of x [..., K] @ w[V, K].T, and the
    log of its sum of exponentials, which the backward takes.  targets (int32, int64, or fp32 as gpt.c has them): a row whose
    target is outside 0 .. V - 1 has a loss of 0."""
    return _calls().linear_xent_forward(x, w, targets, _raw(stream))


def linear_xent_backward(g, x, w, targets, lse, dw=None, want_dx=True, stream=None):
    """Gradients of sum(g * losses): returns dx, of the type of x (None when want_dx is false), and adds to dw (skipped when
    None), which is like w.  g is fp32, one value or one for each row.  Rows without a target have no part in either."""
    return _calls().linear_xent_backward(g, x, w, targets, lse, dw, want_dx, _raw(stream))


# ---------------------------------------------------------------------------------------------
# Generation: a paged key/value cache with the attention that reads it (include/attn_sm100.h), and the draw of the next
# token (include/xent_sm100.h).  The reference's infer_gpt.c:341-408 has no cache and draws on the host.
#
# A layer's cache is k_pages and v_pages [pages, kv_heads, page_size, head_size], fp32 or bf16.  A step brings rows of several
# sequences, one behind the other: page_table [sequences, pages], cu_seqlens [sequences + 1] (first row of each, and the
# end) and past [sequences] (positions before the step) are int32 tensors beside them.  These calls are not differentiable:
# their results are cut off from autograd, whatever their arguments require.
# ---------------------------------------------------------------------------------------------
def paged_append(qkv, k_pages, v_pages, page_table, cu_seqlens, past, rotary=None, rotary_pairs: bool = False, stream=None):
    """Stores the keys and values of qkv [tokens, (n_heads + 2 kv_heads) * head_size] in their sequences' pages and returns the
    queries [tokens, n_heads * head_size]: a view of qkv, or with `rotary` (see rotary_table) a tensor of queries rotated by
    their positions, as the stored keys are.  Columns i and i + R/2 of a head make a pair, or 2i and 2i + 1 with rotary_pairs.
    Not differentiable."""
    return _calls().paged_append(qkv, k_pages, v_pages, page_table, cu_seqlens, past, rotary, rotary_pairs, _raw(stream))


def paged_attention(q, k_pages, v_pages, page_table, cu_seqlens, past, max_new: int = 0, scale=None, out=None, stream=None):
    """Causal attention of q [tokens, n_heads * head_size] over the pages, the new tokens' own keys among them.  `max_new`: the
    largest number of new tokens of a sequence, 0 where the program does not know it; `scale`: head_size ** -0.5 if None.
    Rows behind the last sequence are not written.  Not differentiable."""
    return _calls().paged_attention(q, k_pages, v_pages, page_table, cu_seqlens, past, max_new, scale, out, _raw(stream))


def rotary_table(positions: int, dim: int, base: float = 10000.0, device="cuda"):
    """The table [positions, dim] that paged_append takes as `rotary`: cosines, then sines, of position * base ** (-2 i / dim),
    the angles in 64 bits."""
    import torch

    if positions < 1 or dim < 2 or dim % 2:
        raise ValueError("positions must be positive and dim even")
    freq = base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, stream=None):
    """One class (int32) for each row of logits [rows, classes], drawn with u [rows] from [0, 1).  temperature, top_p and min_p
    (fp32) and top_k (int32) have one value a row, or are None: exp((x - max) / temperature) are the weights, the largest top_k
    classes are kept, of these the shortest run with top_p of their weight, of these the ones with min_p of the largest
    weight.  temperature 0 takes the largest logit.  A row with a NaN, or of -inf alone, gives -1."""
    return _calls().sample(logits, u, temperature, top_k, top_p, min_p, _raw(stream))
