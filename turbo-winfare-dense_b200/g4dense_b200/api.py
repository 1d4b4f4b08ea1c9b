"""ctypes bindings of libg4dense_b200.so (include/g4dense/c_api.h, include/g4dense_b200_ops.h).

There is no fallback: if the library is missing, or CUDA is unavailable when a GPU entry
point is called, the call fails loudly.
"""
from __future__ import annotations

import ctypes
import struct
from pathlib import Path

import numpy as np

LIB_PATH = Path(__file__).resolve().parent / "lib" / "libg4dense_b200.so"
_vp = ctypes.c_void_p
_lib = None


def lib():
    """Loads the native library (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise FileNotFoundError(f"{LIB_PATH} is missing: run g4dense_b200.build.build() first")
        L = ctypes.CDLL(str(LIB_PATH))
        L.g4b_last_error.restype = ctypes.c_char_p
        L.g4b_qmat_create.argtypes = [_vp, _vp, _vp, ctypes.c_int, ctypes.c_int, _vp, ctypes.POINTER(_vp)]
        L.g4b_qmat_destroy.argtypes = [_vp]
        L.g4b_qmat_gemm.argtypes = [_vp, _vp, ctypes.c_int, ctypes.c_int, _vp, ctypes.c_int, _vp]
        L.g4b_qmat_prepare_input.argtypes = [_vp, _vp, ctypes.c_int, ctypes.c_int, _vp]
        L.g4b_qmat_run.argtypes = [_vp, ctypes.c_int, _vp, ctypes.c_int, _vp]
        L.g4b_qmat_info.argtypes = [_vp, _vp]
        L.g4b_qmat_run_partial.argtypes = [_vp, ctypes.c_int, _vp]
        L.g4b_qmat_run_noalloc.argtypes = [_vp, ctypes.c_int, _vp, ctypes.c_int, _vp]
        L.g4b_gemv_int8.argtypes = [_vp, _vp, _vp, _vp, _vp, ctypes.c_int, ctypes.c_int, _vp]
        L.g4b_attn_gate.argtypes = [_vp, _vp, _vp] + [ctypes.c_int] * 5 + [_vp]
        L.g4b_qmat_check_error.argtypes = [_vp]
        _bind_tree(L)
        _bind_engine(L)
        _lib = L
    return _lib


# The argument structs of the tree-verification operators (include/g4dense_b200_ops.h), packed in one
# go: these calls are short, and setting ctypes fields one by one would cost more than the launch.
_TREE_ATTENTION = struct.Struct("@12PN4q12if4x")  # g4b_tree_attention_args
_PAGE_POOL = struct.Struct("@P2q4i")            # g4b_page_pool
_PAGE_TABLES = struct.Struct("@6P4i")           # g4b_page_tables


def _bind_tree(L):
    """Binds the tree-verification and paged-cache operators (include/g4dense_b200_ops.h)."""
    i, i64 = ctypes.c_int, ctypes.c_int64
    args = pool = tables = ctypes.c_char_p  # a packed struct
    L.g4b_tree_attention_workspace.restype = ctypes.c_size_t
    L.g4b_tree_attention_workspace.argtypes = [i, i, i, i]
    L.g4b_tree_attention.argtypes = [args, _vp]
    L.g4b_tree_attention_check_error.argtypes = []
    L.g4b_sample_rows.argtypes = [_vp, i, i, i, i64] + [_vp] * 9
    L.g4b_tree_accept.argtypes = [_vp] * 4 + [i, i, _vp, i, _vp, _vp, _vp]
    L.g4b_pages_reserve.argtypes = [tables, _vp, _vp, _vp]
    L.g4b_pages_fork.argtypes = [pool, tables, _vp, _vp, i, _vp, _vp]
    L.g4b_pages_free.argtypes = [tables, _vp, i, _vp]
    L.g4b_pages_compact.argtypes = [pool, tables, _vp, _vp]
    L.g4b_pages_copy.argtypes = [pool, pool, _vp, _vp, i, _vp]
    L.g4b_pages_commit.argtypes = [pool, _vp, i, _vp, i, _vp, i64, i, _vp, _vp, i, _vp, _vp, _vp, _vp]


class EngineConfig(ctypes.Structure):
    """G4DenseEngineConfig (include/g4dense/c_api.h)."""
    _fields_ = [("container_path", ctypes.c_char_p), ("synthetic_preset", ctypes.c_char_p),
                ("synthetic_seed", ctypes.c_ulonglong), ("synthetic_centered", ctypes.c_int),
                ("draft_path", ctypes.c_char_p), ("draft_preset", ctypes.c_char_p),
                ("draft_seed", ctypes.c_ulonglong), ("draft_k", ctypes.c_int), ("max_context", ctypes.c_int),
                ("kv_bf16", ctypes.c_int), ("tp_rank", ctypes.c_int), ("tp_size", ctypes.c_int),
                ("nccl_unique_id", ctypes.c_void_p), ("device", ctypes.c_int),
                ("gate_min_accept", ctypes.c_double), ("gate_window", ctypes.c_int),
                ("tokenizer_path", ctypes.c_char_p)]


TOKEN_CB = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.c_int, ctypes.c_uint, ctypes.c_char_p)


def _bind_engine(L):
    """Binds the engine-level C API (include/g4dense/c_api.h)."""
    L.g4dense_engine_last_error.restype = ctypes.c_char_p
    L.g4dense_engine_create.restype = _vp
    L.g4dense_engine_create.argtypes = [ctypes.c_char_p]
    L.g4dense_engine_create_ex.restype = _vp
    L.g4dense_engine_create_ex.argtypes = [ctypes.POINTER(EngineConfig)]
    L.g4dense_config_default.argtypes = [ctypes.POINTER(EngineConfig)]
    L.g4dense_engine_destroy.argtypes = [_vp]
    L.g4dense_engine_get_telemetry.restype = ctypes.c_char_p
    L.g4dense_engine_get_telemetry.argtypes = [_vp]
    L.g4dense_options_default.argtypes = [_vp]
    L.g4dense_engine_generate.restype = ctypes.c_char_p
    L.g4dense_engine_generate.argtypes = [_vp, ctypes.c_char_p, ctypes.c_int]
    L.g4dense_engine_generate_ex.restype = ctypes.c_char_p
    L.g4dense_engine_generate_ex.argtypes = [_vp, ctypes.c_char_p, _vp, TOKEN_CB, _vp]
    L.g4dense_engine_generate_text.restype = ctypes.c_char_p
    L.g4dense_engine_generate_text.argtypes = [_vp, ctypes.c_char_p, ctypes.c_int, _vp, TOKEN_CB, _vp]
    L.g4dense_engine_generate_tokens.restype = ctypes.c_char_p
    L.g4dense_engine_generate_tokens.argtypes = [_vp, _vp, ctypes.c_int, _vp, TOKEN_CB, _vp]
    L.g4dense_engine_last_tokens.argtypes = [_vp, _vp, ctypes.c_int]
    L.g4dense_engine_last_rounds.argtypes = [_vp, _vp, ctypes.c_int]
    L.g4dense_engine_forward_batch.argtypes = [_vp, _vp, ctypes.c_int, ctypes.c_int, _vp, ctypes.c_int]
    L.g4dense_engine_set_decode_options.argtypes = [_vp, ctypes.c_longlong, ctypes.c_int, _vp, ctypes.c_int,
                                                    ctypes.c_double, ctypes.c_ulonglong]
    L.g4dense_engine_set_device_sampling.argtypes = [_vp, ctypes.c_int]
    L.g4dense_engine_mtp_draft.argtypes = [_vp, ctypes.c_uint, ctypes.c_int, ctypes.c_int, ctypes.c_int, _vp, _vp]
    L.g4dense_engine_draft_steps.argtypes = [_vp, ctypes.c_uint, ctypes.c_int, ctypes.c_int, _vp, _vp]
    L.g4b_sample_workspace.restype = ctypes.c_size_t
    L.g4b_sample_token.argtypes = [_vp, ctypes.c_int, ctypes.c_float, ctypes.c_float, ctypes.c_int,
                                   ctypes.c_uint64, _vp, _vp, _vp]
    L.g4dense_engine_last_stop_reason.argtypes = [_vp]
    L.g4dense_engine_switch_tier.argtypes = [_vp, ctypes.c_int]
    L.g4dense_engine_stop.argtypes = [_vp]
    L.g4dense_nccl_unique_id.argtypes = [_vp]
    L.g4dense_engine_last_stats.argtypes = [_vp, _vp, ctypes.c_int]
    L.g4dense_engine_set_gate.argtypes = [_vp, ctypes.c_double, ctypes.c_int]
    L.g4dense_engine_time_pass.restype = ctypes.c_double
    L.g4dense_engine_time_pass.argtypes = [_vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    _sz = ctypes.POINTER(ctypes.c_size_t)
    L.g4dense_tokenizer_open.restype = _vp
    L.g4dense_tokenizer_open.argtypes = [ctypes.c_char_p, ctypes.c_int]
    L.g4dense_engine_tokenizer.restype = _vp
    L.g4dense_engine_tokenizer.argtypes = [_vp]
    L.g4dense_tokenizer_destroy.argtypes = [_vp]
    L.g4dense_tokenizer_encode.argtypes = [_vp, ctypes.c_char_p, ctypes.c_size_t, ctypes.c_int, _vp, ctypes.c_int]
    L.g4dense_tokenizer_decode.restype = _vp
    L.g4dense_tokenizer_decode.argtypes = [_vp, _vp, ctypes.c_int, ctypes.c_int, _sz]
    L.g4dense_tokenizer_decode_single.restype = _vp
    L.g4dense_tokenizer_decode_single.argtypes = [_vp, ctypes.c_uint, ctypes.c_int, _sz]
    L.g4dense_tokenizer_chat_template.restype = ctypes.c_char_p
    L.g4dense_tokenizer_chat_template.argtypes = [_vp, ctypes.c_char_p]
    L.g4dense_tokenizer_special_ids.argtypes = [_vp, _vp]
    L.g4dense_tokenizer_stop_ids.argtypes = [_vp, _vp, ctypes.c_int]
    L.g4dense_tokenizer_byte_value.argtypes = [_vp, ctypes.c_uint, ctypes.POINTER(ctypes.c_ubyte)]
    L.g4dense_tokenizer_is_special.argtypes = [_vp, ctypes.c_uint]
    L.g4dense_detokenizer_create.restype = _vp
    L.g4dense_detokenizer_create.argtypes = [_vp, ctypes.c_int]
    L.g4dense_detokenizer_push.restype = _vp
    L.g4dense_detokenizer_push.argtypes = [_vp, ctypes.c_uint, _sz]
    L.g4dense_detokenizer_finish.restype = _vp
    L.g4dense_detokenizer_finish.argtypes = [_vp, _sz]
    L.g4dense_detokenizer_destroy.argtypes = [_vp]
    L.g4dense_stop_matcher_create.restype = _vp
    L.g4dense_stop_matcher_create.argtypes = [ctypes.POINTER(ctypes.c_char_p), ctypes.c_int]
    L.g4dense_stop_matcher_push.restype = _vp
    L.g4dense_stop_matcher_push.argtypes = [_vp, ctypes.c_char_p, ctypes.c_size_t, _sz]
    L.g4dense_stop_matcher_finish.restype = _vp
    L.g4dense_stop_matcher_finish.argtypes = [_vp, _sz]
    L.g4dense_stop_matcher_stopped.argtypes = [_vp, ctypes.POINTER(ctypes.c_char_p)]
    L.g4dense_stop_matcher_destroy.argtypes = [_vp]
    L.g4dense_utf8_repair.restype = _vp
    L.g4dense_utf8_repair.argtypes = [ctypes.c_char_p, ctypes.c_size_t, ctypes.c_int, _sz, _sz]
    L.g4dense_container_validate.argtypes = [ctypes.c_char_p]
    L.g4dense_engine_profile_gemms.restype = ctypes.c_double
    L.g4dense_engine_profile_gemms.argtypes = [_vp, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_ulonglong),
                                               ctypes.POINTER(ctypes.c_int)]


def _check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} failed ({rc}): {lib().g4b_last_error().decode()}")


def _dptr(t):
    """Device pointer of a torch CUDA tensor."""
    return ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    return ctypes.c_void_p(stream.cuda_stream if stream is not None else 0)


def gemv_int8(W, S, B, x, out, stream=None):
    """out[r] = sum_k (W[r][k] * s + b) * x[k]: W uint8 [rows][K], S/B bf16 bits [rows][K/64],
    x fp32 [K], out fp32 [rows] (torch CUDA tensors)."""
    _check(lib().g4b_gemv_int8(_dptr(W), _dptr(S), _dptr(B), _dptr(x), _dptr(out), W.shape[0], W.shape[1],
                               _stream(stream)), "g4b_gemv_int8")


def attn_gate(ctx, gate, out, stream=None):
    """out = ctx * sigmoid(gate) over [batch][n] fp32 torch CUDA tensors (row strides honoured)."""
    _check(lib().g4b_attn_gate(_dptr(ctx), _dptr(gate), _dptr(out), ctx.shape[1], ctx.shape[0], ctx.stride(0),
                               gate.stride(0), out.stride(0), _stream(stream)), "g4b_attn_gate")


def sample_workspace_bytes():
    return int(lib().g4b_sample_workspace())


def sample_token(logits, temperature, top_p, top_k, seed, workspace, out, stream=None):
    """Draws a token from the fp32 logits row (torch CUDA tensor) into out (uint32/int32 CUDA
    tensor of one element) as the reference's sample_token does; workspace is a CUDA byte tensor
    of sample_workspace_bytes()."""
    _check(lib().g4b_sample_token(_dptr(logits), logits.numel(), temperature, top_p, top_k, seed & (2**64 - 1),
                                  _dptr(workspace), _dptr(out), _stream(stream)), "g4b_sample_token")

_dtypes = {}  # torch dtype -> g4b_dtype, filled by _types()
_i32 = _f32 = _here = _stream_of = None


def _types():
    """Loads torch's types and the library once; returns the library."""
    global _i32, _f32, _here, _stream_of
    if _i32 is None:
        import torch
        _dtypes.update({torch.bfloat16: 0, torch.float16: 1, torch.float32: 2})
        _f32 = torch.float32
        # The current device, on which every tensor of a call has to be (kernels launch there), and the handle
        # of its current stream: torch.cuda.current_stream() makes an object of it, 3 us a call.
        _here = torch.cuda.current_device
        _stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
        _i32 = torch.int32
    return lib()


def _bad(what):
    raise ValueError(what)


def _ints(name, t, n, dev):
    """Device pointer of a contiguous int32 tensor of n elements on device `dev`."""
    if t.dtype is not _i32 or t.get_device() != dev or t.numel() != n or not t.is_contiguous():
        _bad(f"{name}: a contiguous int32 CUDA tensor of {n} elements on the current device, {dev}, is needed, got "
             f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _floats(name, t, n, dev):
    """As _ints for float32; None stays None."""
    if t is None:
        return None
    if t.dtype is not _f32 or t.get_device() != dev or t.numel() != n or not t.is_contiguous():
        _bad(f"{name}: a contiguous float32 CUDA tensor of {n} elements on the current device, {dev}, is needed, got "
             f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows_of(name, t, dtype, shape, dev):
    """(device pointer, stride of the first dimension) of a tensor on device `dev`, contiguous but for that one."""
    if t.dtype is not dtype or t.get_device() != dev or t.shape != shape:
        _bad(f"{name}: a {dtype} CUDA tensor of shape {tuple(shape)} on the current device, {dev}, is needed, got "
             f"{t.dtype} {tuple(t.shape)} on {t.device}")
    n, strides = 1, t.stride()
    for k in range(len(shape) - 1, 0, -1):
        if strides[k] != n and shape[k] != 1:
            _bad(f"{name} has to be contiguous but for its first dimension")
        n *= shape[k]
    return t.data_ptr(), strides[0] if shape[0] > 1 else n


def _at(stream, dev):
    """Handle of the stream given, else of torch's current one: what made the inputs is ordered before."""
    return _stream_of(dev) if stream is None else stream.cuda_stream


def tree_mask(parents, words=None):
    """Mask words and depths of one tree from its parents (parents[i] < i, -1 for a root): (mask
    [n][words] int32, depth [n] int32) numpy arrays for tree_attention, node i seeing itself and its
    ancestors."""
    n = len(parents)
    words = words or max(1, (n + 31) // 32)
    mask, depth = np.zeros((n, words), np.uint32), np.zeros(n, np.int32)
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            _bad(f"tree_mask: parent {p} of node {i}")
        if p >= 0:
            mask[i] = mask[p]
            depth[i] = depth[p] + 1
        mask[i, i // 32] |= np.uint32(1 << (i % 32))
    return mask.view(np.int32), depth


def tree_attention_workspace(max_nodes, heads, kv_heads, head_dim):
    """Bytes of workspace tree_attention needs (ValueError for a shape it does not support)."""
    n = int(lib().g4b_tree_attention_workspace(max_nodes, heads, kv_heads, head_dim))
    if not n:
        _bad(f"tree_attention: max_nodes {max_nodes} (1..256), heads {heads} (a multiple of {kv_heads}), head_dim "
             f"{head_dim} (64, 128, 256 or 512)")
    return n


def tree_attention(q, k_pool, v_pool, table, lens, k_new, v_new, cu_nodes, mask, out, workspace, *, max_nodes, scale,
                   depth=None, window=0, stream=None):
    """Attention of drafted-token trees over a paged K/V cache (g4b_tree_attention). q, out
    [tokens][heads][dim]; k_pool, v_pool [pages][page_size][kv_heads][dim]; k_new, v_new
    [tokens][kv_heads][dim], all bf16 or all fp16 torch CUDA tensors (token and page strides
    honoured); table [seqs][width], lens [seqs], cu_nodes [seqs + 1], mask [tokens][words], depth
    [tokens] int32; workspace a byte tensor of tree_attention_workspace()."""
    L, dev = _types(), _here()
    shape, pool, dtype = q.shape, k_pool.shape, q.dtype
    if len(shape) != 3 or len(pool) != 4 or _dtypes.get(dtype, 2) > 1:
        _bad(f"tree_attention: q [tokens][heads][dim] and pools [pages][page_size][kv_heads][dim] of dtype bfloat16 or "
             f"float16 are needed, got {tuple(shape)}, {tuple(pool)}, {dtype}")
    tokens, heads, dim = shape
    pages, page_size, kv_heads, _ = pool
    new = (tokens, kv_heads, dim)
    if pool[3] != dim:
        _bad("tree_attention: q and the pools differ in head_dim")
    pq, q_stride = _rows_of("q", q, dtype, shape, dev)
    po, out_stride = _rows_of("out", out, dtype, shape, dev)
    pk, page_stride = _rows_of("k_pool", k_pool, dtype, pool, dev)
    pv, v_stride = _rows_of("v_pool", v_pool, dtype, pool, dev)
    pkn, new_stride = _rows_of("k_new", k_new, dtype, new, dev)
    pvn, vn_stride = _rows_of("v_new", v_new, dtype, new, dev)
    if v_stride != page_stride or vn_stride != new_stride:
        _bad("tree_attention: K and V differ in their strides")
    if window and depth is None:
        _bad("tree_attention: a window needs the nodes' depths")
    seqs, width, words = lens.numel(), table.shape[-1], mask.shape[-1]
    if workspace.get_device() != dev or not workspace.is_contiguous():
        _bad(f"workspace: a contiguous CUDA tensor on the current device, {dev}, is needed")
    a = _TREE_ATTENTION.pack(
        pq, pk, pv, pkn, pvn, po, _ints("table", table, seqs * width, dev), _ints("lens", lens, seqs, dev),
        _ints("cu_nodes", cu_nodes, seqs + 1, dev), _ints("mask", mask, tokens * words, dev),
        0 if depth is None else _ints("depth", depth, tokens, dev), workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), q_stride, out_stride, new_stride, page_stride, seqs, tokens,
        max_nodes, pages, page_size, width, words, heads, kv_heads, dim, window, _dtypes[dtype], scale)
    rc = L.g4b_tree_attention(a, _at(stream, dev))
    if rc:
        _check(rc, "g4b_tree_attention")


def tree_attention_check_error():
    """Synchronizes; raises when a tree_attention launch hit a bounded-wait timeout."""
    _check(lib().g4b_tree_attention_check_error(), "g4b_tree_attention_check_error")


def sample_rows(logits, uniform, token, prob=None, kept=None, temperature=None, top_k=None, top_p=None, min_p=None,
                stream=None):
    """One token per row of logits [rows][vocab] (bf16, fp16 or fp32; row stride honoured) into token
    [rows] int32, from uniform [rows] float32 in [0, 1), with per-row temperature, top_p, min_p
    (float32) and top_k (int32) where given (g4b_sample_rows). prob [rows] float32 and kept [rows]
    int32 receive the token's share of the kept mass and the number of kept entries."""
    L, dev = _types(), _here()
    if logits.dim() != 2 or logits.dtype not in _dtypes:
        _bad(f"sample_rows: logits [rows][vocab] of dtype bfloat16, float16 or float32 are needed, got "
             f"{tuple(logits.shape)} {logits.dtype}")
    if uniform is None:
        _bad("sample_rows: uniform numbers are needed")
    rows, vocab = logits.shape
    ptr, stride = _rows_of("logits", logits, logits.dtype, logits.shape, dev)
    rc = L.g4b_sample_rows(ptr, _dtypes[logits.dtype], rows, vocab, stride, _floats("uniform", uniform, rows, dev),
                           _floats("temperature", temperature, rows, dev), None if top_k is None else _ints("top_k", top_k, rows, dev),
                           _floats("top_p", top_p, rows, dev), _floats("min_p", min_p, rows, dev), _ints("token", token, rows, dev),
                           _floats("prob", prob, rows, dev), None if kept is None else _ints("kept", kept, rows, dev), _at(stream, dev))
    if rc:
        _check(rc, "g4b_sample_rows")


def tree_accept(tokens, parents, sampled, cu_nodes, path, count, next_token, stream=None):
    """Walks each tree along the drawn tokens (g4b_tree_accept): path [seqs][width], count [seqs] and
    next_token [seqs] from tokens, parents, sampled [nodes] and cu_nodes [seqs + 1], all int32."""
    L, dev = _types(), _here()
    n, seqs, width = tokens.numel(), cu_nodes.numel() - 1, path.shape[-1]
    rc = L.g4b_tree_accept(_ints("tokens", tokens, n, dev), _ints("parents", parents, n, dev), _ints("sampled", sampled, n, dev),
                           _ints("cu_nodes", cu_nodes, seqs + 1, dev), seqs, n, _ints("path", path, seqs * width, dev), width,
                           _ints("count", count, seqs, dev), _ints("next_token", next_token, seqs, dev), _at(stream, dev))
    if rc:
        _check(rc, "g4b_tree_accept")


def _pool(pool, dev):
    """Packed g4b_page_pool of a CUDA tensor [planes][pages][page_size][...] with contiguous pages."""
    shape, strides, size = pool.shape, pool.stride(), pool.element_size()
    if pool.get_device() != dev or len(shape) < 4:
        _bad(f"pool: a CUDA tensor [planes][pages][page_size][row...] on the current device, {dev}, is needed")
    n = 1
    for k in range(len(shape) - 1, 1, -1):
        if strides[k] != n and shape[k] != 1:
            _bad("pool: the rows of a page have to be contiguous")
        n *= shape[k]
    page = (strides[1] if shape[1] > 1 else n) * size
    plane = (strides[0] if shape[0] > 1 else shape[1] * n) * size
    return _PAGE_POOL.pack(pool.data_ptr(), plane, page, shape[0], shape[1], shape[2], n // max(shape[2], 1) * size)


def _tables(refs, table, lens, refs_out, table_out, lens_out, page_size, dev):
    pages, (seqs, width) = refs.numel(), table.shape
    return _PAGE_TABLES.pack(
        _ints("refs", refs, pages, dev), _ints("table", table, seqs * width, dev), 0 if lens is None else _ints("lens", lens, seqs, dev),
        _ints("refs_out", refs_out, pages, dev), _ints("table_out", table_out, seqs * width, dev),
        0 if lens_out is None else _ints("lens_out", lens_out, seqs, dev), pages, seqs, width, page_size)


def pages_reserve(refs, table, lens, grow, page_size, refs_out, table_out, status, stream=None):
    """Pages for grow[s] more tokens of every sequence (g4b_pages_reserve). int32 CUDA tensors: refs
    [pages], table [seqs][width], lens, grow [seqs], status [1]; the outputs may be the inputs."""
    L, dev = _types(), _here()
    rc = L.g4b_pages_reserve(_tables(refs, table, lens, refs_out, table_out, None, page_size, dev),
                             _ints("grow", grow, lens.numel(), dev), _ints("status", status, 1, dev), _at(stream, dev))
    if rc:
        _check(rc, "g4b_pages_reserve")


def pages_fork(pool, refs, table, lens, src, dst, refs_out, table_out, lens_out, status, stream=None):
    """Sequences dst[i] become continuations of src[i] (g4b_pages_fork): full pages shared, a partial
    last page copied. pool [planes][pages][page_size][row...]."""
    L, dev, n = _types(), _here(), src.numel()
    rc = L.g4b_pages_fork(_pool(pool, dev), _tables(refs, table, lens, refs_out, table_out, lens_out, pool.shape[2], dev),
                          _ints("src", src, n, dev), _ints("dst", dst, n, dev), n, _ints("status", status, 1, dev), _at(stream, dev))
    if rc:
        _check(rc, "g4b_pages_fork")


def pages_free(refs, table, lens, seqs, page_size, refs_out, table_out, lens_out, stream=None):
    """Releases the pages of the sequences seqs[] and empties them (g4b_pages_free)."""
    L, dev, n = _types(), _here(), seqs.numel()
    rc = L.g4b_pages_free(_tables(refs, table, lens, refs_out, table_out, lens_out, page_size, dev), _ints("seqs", seqs, n, dev), n,
                          _at(stream, dev))
    if rc:
        _check(rc, "g4b_pages_free")


def pages_compact(pool, refs, table, refs_out, table_out, moves, stream=None):
    """Moves live pages to the front of the pool (g4b_pages_compact); moves [1 + 2 * pages] int32
    receives their number and the (from, to) pairs."""
    L, dev = _types(), _here()
    rc = L.g4b_pages_compact(_pool(pool, dev), _tables(refs, table, None, refs_out, table_out, None, pool.shape[2], dev),
                             _ints("moves", moves, 1 + 2 * refs.numel(), dev), _at(stream, dev))
    if rc:
        _check(rc, "g4b_pages_compact")


def pages_copy(pool, to_pool, src, dst, stream=None):
    """Page src[i] of pool to page dst[i] of to_pool, in every plane (g4b_pages_copy)."""
    L, dev, n = _types(), _here(), src.numel()
    rc = L.g4b_pages_copy(_pool(pool, dev), _pool(to_pool, dev), _ints("src", src, n, dev), _ints("dst", dst, n, dev), n, _at(stream, dev))
    if rc:
        _check(rc, "g4b_pages_copy")


def pages_commit(pool, table, lens, rows, cu_nodes, path, count, lens_out, status=None, stream=None):
    """Writes the accepted nodes' rows [planes][tokens][row...] into their sequences' pages and the
    new lengths into lens_out (g4b_pages_commit). path None: the first count[s] rows."""
    L, dev = _types(), _here()
    shape, want, seqs, width = rows.shape, pool.shape, lens.numel(), table.shape[-1]
    tokens = shape[1]
    if len(shape) != len(want) - 1 or shape[0] != want[0] or shape[2:] != want[3:]:
        _bad("pages_commit: rows have to be [planes][tokens][row...] like the pool")
    ptr, stride = _rows_of("rows", rows, pool.dtype, shape, dev)
    rc = L.g4b_pages_commit(_pool(pool, dev), _ints("table", table, seqs * width, dev), width, _ints("lens", lens, seqs, dev), seqs, ptr,
                            stride * rows.element_size(), tokens, _ints("cu_nodes", cu_nodes, seqs + 1, dev),
                            None if path is None else _ints("path", path, seqs * path.shape[-1], dev),
                            0 if path is None else path.shape[-1], _ints("count", count, seqs, dev),
                            None if status is None else _ints("status", status, 1, dev), _ints("lens_out", lens_out, seqs, dev),
                            _at(stream, dev))
    if rc:
        _check(rc, "g4b_pages_commit")


class QMat:
    """A prepared INT4 G64 matrix on the device (g4b_qmat)."""

    def __init__(self, W, S, B, stream=None):
        """W, S, B: torch CUDA tensors in container layout (int32/uint32 [N][K/8],
        int16/uint16 [N][K/64] x2)."""
        self.N = W.shape[0]
        self.K = W.shape[1] * 8
        h = ctypes.c_void_p()
        _check(lib().g4b_qmat_create(_dptr(W), _dptr(S), _dptr(B), self.N, self.K, _stream(stream),
                                     ctypes.byref(h)), "g4b_qmat_create")
        self.h = h

    def gemm(self, x, out, stream=None):
        _check(lib().g4b_qmat_gemm(self.h, _dptr(x), x.shape[1], x.shape[0], _dptr(out), out.shape[1],
                                   _stream(stream)), "g4b_qmat_gemm")

    def prepare(self, x, stream=None):
        _check(lib().g4b_qmat_prepare_input(self.h, _dptr(x), x.shape[1], x.shape[0], _stream(stream)),
               "g4b_qmat_prepare_input")

    def run(self, M, out, stream=None):
        _check(lib().g4b_qmat_run(self.h, M, _dptr(out), out.shape[1], _stream(stream)), "g4b_qmat_run")

    def run_noalloc(self, M, out, stream=None):
        """g4b_qmat_run with the library's static split-K scratch (allocates nothing)."""
        _check(lib().g4b_qmat_run_noalloc(self.h, M, _dptr(out), out.shape[1], _stream(stream)),
               "g4b_qmat_run_noalloc")

    def run_partial(self, M, stream=None):
        _check(lib().g4b_qmat_run_partial(self.h, M, _stream(stream)), "g4b_qmat_run_partial")

    def check_error(self):
        _check(lib().g4b_qmat_check_error(self.h), "g4b_qmat_check_error")

    def info(self):
        o = np.zeros(4, np.int32)
        _check(lib().g4b_qmat_info(self.h, o.ctypes.data_as(_vp)), "g4b_qmat_info")
        return {"N": int(o[0]), "K": int(o[1]), "grid_m5": int(o[2]), "max_slots": int(o[3])}

    def close(self):
        if getattr(self, "h", None):
            lib().g4b_qmat_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class GenOptions(ctypes.Structure):
    """G4DenseGenerationOptions (include/g4dense/c_api.h:24-36)."""
    _fields_ = [("max_tokens", ctypes.c_int), ("temperature", ctypes.c_float), ("top_p", ctypes.c_float),
                ("top_k", ctypes.c_int), ("repetition_penalty", ctypes.c_float), ("has_seed", ctypes.c_int),
                ("seed", ctypes.c_ulonglong), ("system_prompt", ctypes.c_char_p),
                ("stop_strings", ctypes.c_void_p), ("stop_count", ctypes.c_int), ("tier_id", ctypes.c_int)]


def _eng_err(what):
    raise RuntimeError(f"{what}: {lib().g4dense_engine_last_error().decode()}")


class Engine:
    """The engine behind include/g4dense/c_api.h (greedy or sampled, optional drafter)."""

    def __init__(self, target=None, preset=None, seed=0, centered=False, draft=None, draft_preset=None,
                 draft_seed=1, draft_k=0, max_context=4096, kv_bf16=False, tp_rank=0, tp_size=1,
                 nccl_id=None, device=-1, gate_min_accept=0.45, gate_window=24, tokenizer_path=None):
        L = lib()
        cfg = EngineConfig()
        L.g4dense_config_default(ctypes.byref(cfg))
        self._keep = []
        def cstr(x):
            if x is None:
                return None
            b = str(x).encode()
            self._keep.append(b)
            return b
        cfg.container_path = cstr(target)
        cfg.synthetic_preset = cstr(preset)
        cfg.synthetic_seed = seed
        cfg.synthetic_centered = 1 if centered else 0
        cfg.draft_path = cstr(draft)
        cfg.draft_preset = cstr(draft_preset)
        cfg.draft_seed = draft_seed
        cfg.draft_k = draft_k
        cfg.max_context = max_context
        cfg.kv_bf16 = 1 if kv_bf16 else 0
        cfg.tp_rank, cfg.tp_size = tp_rank, tp_size
        if nccl_id is not None:
            self._nid = ctypes.create_string_buffer(bytes(nccl_id), 128)
            cfg.nccl_unique_id = ctypes.cast(self._nid, ctypes.c_void_p)
        cfg.device = device
        cfg.gate_min_accept = gate_min_accept
        cfg.gate_window = gate_window
        cfg.tokenizer_path = cstr(tokenizer_path)
        self.h = L.g4dense_engine_create_ex(ctypes.byref(cfg))
        if not self.h:
            _eng_err("g4dense_engine_create_ex")

    def set_decode_options(self, stop_token=-1, draft_k=-1, replay=None, mismatch_rate=0.0, mismatch_seed=0):
        r = None if replay is None else np.ascontiguousarray(replay, np.uint32)
        if lib().g4dense_engine_set_decode_options(self.h, stop_token, draft_k,
                                                   None if r is None else r.ctypes.data_as(_vp),
                                                   0 if r is None else len(r), mismatch_rate, mismatch_seed):
            _eng_err("g4dense_engine_set_decode_options")

    def set_device_sampling(self, on):
        if lib().g4dense_engine_set_device_sampling(self.h, 1 if on else 0):
            _eng_err("g4dense_engine_set_device_sampling")

    def generate(self, prompt, max_tokens, temperature=0.0, top_p=1.0, top_k=0, seed=None, callback=None,
                 repetition_penalty=1.0):
        o = GenOptions()
        lib().g4dense_options_default(ctypes.byref(o))
        o.max_tokens = max_tokens
        o.temperature, o.top_p, o.top_k = temperature, top_p, top_k
        o.repetition_penalty = repetition_penalty
        o.has_seed = 0 if seed is None else 1
        o.seed = 0 if seed is None else seed
        p = np.ascontiguousarray(prompt, np.uint32)
        cb = TOKEN_CB(lambda u, i, t, d: int(callback(t)) if callback else 1)
        r = lib().g4dense_engine_generate_tokens(self.h, p.ctypes.data_as(_vp), len(p), ctypes.byref(o), cb, None)
        if r is None:
            _eng_err("g4dense_engine_generate_tokens")
        out = np.zeros(max_tokens + 32, np.uint32)
        n = lib().g4dense_engine_last_tokens(self.h, out.ctypes.data_as(_vp), len(out))
        return out[:n].copy()

    def generate_text(self, prompt, use_chat_template=True, max_tokens=512, temperature=0.0, top_p=1.0, top_k=0,
                      seed=None, callback=None, options=None):
        """ForwardRunner::generate(prompt, options) through g4dense_engine_generate_text: returns the
        concatenated pieces (bytes); callback(token, piece_bytes) -> bool continues. `options`
        (a GenOptions) overrides the keyword sampling arguments."""
        o = options
        if o is None:
            o = GenOptions()
            lib().g4dense_options_default(ctypes.byref(o))
            o.max_tokens = max_tokens
            o.temperature, o.top_p, o.top_k = temperature, top_p, top_k
            o.has_seed = 0 if seed is None else 1
            o.seed = 0 if seed is None else seed
        cb = TOKEN_CB(lambda u, i, t, d: int(callback(t, d)) if callback else 1)
        r = lib().g4dense_engine_generate_text(self.h, _as_bytes(prompt), 1 if use_chat_template else 0,
                                               ctypes.byref(o), cb, None)
        if r is None:
            _eng_err("g4dense_engine_generate_text")
        return r

    def tokens(self, cap=1 << 16):
        out = np.zeros(cap, np.uint32)
        n = lib().g4dense_engine_last_tokens(self.h, out.ctypes.data_as(_vp), cap)
        return out[:n].copy()

    def tokenizer(self):
        """The engine's own tokenizer (None when it loaded none)."""
        t = lib().g4dense_engine_tokenizer(self.h)
        return Tokenizer(_handle=t, _owner=self) if t else None

    def rounds(self, cap=4096):
        buf = np.zeros(3 * cap, np.int32)
        n = lib().g4dense_engine_last_rounds(self.h, buf.ctypes.data_as(_vp), cap)
        return [tuple(int(v) for v in buf[3 * i:3 * i + 3]) for i in range(n)]

    def forward_batch(self, tokens, base, vocab=None, all_positions=True):
        t = np.ascontiguousarray(tokens, np.uint32)
        out = None
        if vocab is not None:
            out = np.zeros((len(t) if all_positions else 1, vocab), np.float32)
        rc = lib().g4dense_engine_forward_batch(self.h, t.ctypes.data_as(_vp), len(t), base,
                                                None if out is None else out.ctypes.data_as(_vp),
                                                1 if all_positions else 0)
        if rc:
            _eng_err("g4dense_engine_forward_batch")
        return out

    def mtp_draft(self, seed_token, context_length, hidden_row, k, vocab):
        """Greedy MTP drafting from the target's current state: (tokens [k], logits [k][vocab])."""
        toks = np.zeros(k, np.uint32)
        logits = np.zeros((k, vocab), np.float32)
        if lib().g4dense_engine_mtp_draft(self.h, seed_token, context_length, hidden_row, k,
                                          toks.ctypes.data_as(_vp), logits.ctypes.data_as(_vp)):
            _eng_err("g4dense_engine_mtp_draft")
        return toks, logits

    def draft_steps(self, token, pos, k, vocab=None):
        """Greedy drafting by the separate drafter: k chained one-row steps from `token` at position
        `pos` -> (tokens [k], logits [k][vocab] or None)."""
        toks = np.zeros(k, np.uint32)
        logits = None if vocab is None else np.zeros((k, vocab), np.float32)
        if lib().g4dense_engine_draft_steps(self.h, token, pos, k, toks.ctypes.data_as(_vp),
                                            None if logits is None else logits.ctypes.data_as(_vp)):
            _eng_err("g4dense_engine_draft_steps")
        return toks, logits

    STAT_KEYS = ("emitted", "decode_gpu_ms", "ttft_ms", "total_ms", "drafted", "accepted", "rounds",
                 "gated_steps", "launches", "h2d_bytes", "d2h_bytes", "decode_wall_ms")

    def stats(self):
        buf = np.zeros(len(self.STAT_KEYS), np.float64)
        n = lib().g4dense_engine_last_stats(self.h, buf.ctypes.data_as(_vp), len(buf))
        return dict(zip(self.STAT_KEYS[:n], buf[:n].tolist()))

    def set_gate(self, min_accept=0.45, window=24):
        if lib().g4dense_engine_set_gate(self.h, min_accept, window):
            _eng_err("g4dense_engine_set_gate")

    def time_pass(self, which, batch, reps=5, pos=0):
        ms = lib().g4dense_engine_time_pass(self.h, which, batch, pos, reps)
        if ms < 0:
            _eng_err("g4dense_engine_time_pass")
        return ms

    def profile_gemms(self, batch, reps=3):
        b = ctypes.c_ulonglong(0)
        n = ctypes.c_int(0)
        ms = lib().g4dense_engine_profile_gemms(self.h, batch, reps, ctypes.byref(b), ctypes.byref(n))
        if ms < 0:
            _eng_err("g4dense_engine_profile_gemms")
        return ms, int(b.value), int(n.value)

    def telemetry(self):
        import json
        return json.loads(lib().g4dense_engine_get_telemetry(self.h).decode())

    def close(self):
        if getattr(self, "h", None):
            lib().g4dense_engine_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _as_bytes(x):
    return x if isinstance(x, bytes) else str(x).encode()


def _take(ptr, n):
    if not ptr:
        raise RuntimeError(lib().g4dense_engine_last_error().decode())
    return ctypes.string_at(ptr, n.value)


class Tokenizer:
    """The engine's tokenizer (g4dense_tokenizer_*): Gemma-4 tokenizer.json BPE, chat template,
    byte-fallback decoding. Text goes in as str or UTF-8 bytes and comes out as bytes."""

    def __init__(self, path=None, arch=0, _handle=None, _owner=None):
        self._owner = _owner
        if _handle is not None:
            self.h = _handle
            return
        self.h = lib().g4dense_tokenizer_open(None if path is None else str(path).encode(), arch)
        if not self.h:
            _eng_err("g4dense_tokenizer_open")

    def encode(self, text, add_bos=True):
        b = _as_bytes(text)
        n = lib().g4dense_tokenizer_encode(self.h, b, len(b), 1 if add_bos else 0, None, 0)
        if n < 0:
            _eng_err("g4dense_tokenizer_encode")
        out = np.zeros(max(n, 1), np.uint32)
        n = lib().g4dense_tokenizer_encode(self.h, b, len(b), 1 if add_bos else 0, out.ctypes.data_as(_vp), len(out))
        return out[:n].tolist()

    def decode(self, ids, skip_special=True):
        a = np.ascontiguousarray(ids, np.uint32)
        n = ctypes.c_size_t(0)
        return _take(lib().g4dense_tokenizer_decode(self.h, a.ctypes.data_as(_vp), len(a), 1 if skip_special else 0,
                                                    ctypes.byref(n)), n)

    def decode_single(self, tid, skip_special=True):
        n = ctypes.c_size_t(0)
        return _take(lib().g4dense_tokenizer_decode_single(self.h, tid, 1 if skip_special else 0, ctypes.byref(n)), n)

    def chat_template(self, messages):
        """messages: a JSON string, or [(role, content)] / [{"role": .., "content": ..}]."""
        import json
        if not isinstance(messages, (str, bytes)):
            messages = json.dumps([m if isinstance(m, dict) else {"role": m[0], "content": m[1]} for m in messages])
        r = lib().g4dense_tokenizer_chat_template(self.h, _as_bytes(messages))
        if r is None:
            _eng_err("g4dense_tokenizer_chat_template")
        return r

    def special_ids(self):
        v = np.zeros(6, np.uint32)
        lib().g4dense_tokenizer_special_ids(self.h, v.ctypes.data_as(_vp))
        return dict(zip(("bos", "eos", "pad", "unk", "end_of_turn", "vocab_size"), v.tolist()))

    def stop_ids(self):
        v = np.zeros(16, np.uint32)
        n = lib().g4dense_tokenizer_stop_ids(self.h, v.ctypes.data_as(_vp), len(v))
        return v[:n].tolist()

    def byte_value(self, tid):
        b = ctypes.c_ubyte(0)
        return b.value if lib().g4dense_tokenizer_byte_value(self.h, tid, ctypes.byref(b)) else None

    def is_special(self, tid):
        return bool(lib().g4dense_tokenizer_is_special(self.h, tid))

    def detokenizer(self, skip_special=True):
        return Detokenizer(self, skip_special)

    def close(self):
        if getattr(self, "h", None) and self._owner is None:
            lib().g4dense_tokenizer_destroy(self.h)
        self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Detokenizer:
    """IncrementalDetokenizer: push(id) -> bytes now complete; finish() -> the rest."""

    def __init__(self, tok: Tokenizer, skip_special=True):
        self._tok = tok
        self.h = lib().g4dense_detokenizer_create(tok.h, 1 if skip_special else 0)
        if not self.h:
            _eng_err("g4dense_detokenizer_create")

    def push(self, tid):
        n = ctypes.c_size_t(0)
        return _take(lib().g4dense_detokenizer_push(self.h, tid, ctypes.byref(n)), n)

    def finish(self):
        n = ctypes.c_size_t(0)
        return _take(lib().g4dense_detokenizer_finish(self.h, ctypes.byref(n)), n)

    def __del__(self):
        try:
            if self.h:
                lib().g4dense_detokenizer_destroy(self.h)
        except Exception:
            pass


class StopMatcher:
    """StreamingStopMatcher over byte strings."""

    def __init__(self, stops):
        arr = (ctypes.c_char_p * max(1, len(stops)))(*[_as_bytes(s) for s in stops])
        self.h = lib().g4dense_stop_matcher_create(arr, len(stops))
        if not self.h:
            _eng_err("g4dense_stop_matcher_create")

    def push(self, text):
        b = _as_bytes(text)
        n = ctypes.c_size_t(0)
        return _take(lib().g4dense_stop_matcher_push(self.h, b, len(b), ctypes.byref(n)), n)

    def finish(self):
        n = ctypes.c_size_t(0)
        return _take(lib().g4dense_stop_matcher_finish(self.h, ctypes.byref(n)), n)

    @property
    def stopped(self):
        return bool(lib().g4dense_stop_matcher_stopped(self.h, None))

    @property
    def matched(self):
        m = ctypes.c_char_p()
        lib().g4dense_stop_matcher_stopped(self.h, ctypes.byref(m))
        return m.value or b""

    def __del__(self):
        try:
            if self.h:
                lib().g4dense_stop_matcher_destroy(self.h)
        except Exception:
            pass


def utf8_repair(data: bytes, flush_all: bool):
    """-> (repaired bytes, bytes of `data` consumed)."""
    used, n = ctypes.c_size_t(0), ctypes.c_size_t(0)
    p = lib().g4dense_utf8_repair(data, len(data), 1 if flush_all else 0, ctypes.byref(used), ctypes.byref(n))
    return ctypes.string_at(p, n.value), used.value


def validate_container(path) -> str:
    """Checks a container's header against its file with the engine loader's rules (no GPU
    needed). Returns "g4dense" or "g4mtp"; raises ValueError listing every broken rule."""
    rc = lib().g4dense_container_validate(str(path).encode())
    if rc < 0:
        raise ValueError(lib().g4dense_engine_last_error().decode())
    return {1: "g4dense", 2: "g4mtp"}[rc]
