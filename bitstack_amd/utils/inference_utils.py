"""Fused inference helpers with the reference's names and argument meanings
(bitstack/utils/inference_utils.py); every one is a thin call into the C ABI.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from bitstack_amd import _lib


def _f16c(t):
    if t.dtype != torch.float16:
        raise TypeError(f"expected float16, got {t.dtype}")
    return t.contiguous()


def _dims(u, vt):
    if u.dim() != 3 or vt.dim() != 3 or u.shape[0] != vt.shape[0] or u.shape[2] != vt.shape[1]:
        raise ValueError(f"u {tuple(u.shape)} / vt {tuple(vt.shape)} are not [I,M,K] / [I,K,N]")
    I, M, K = u.shape
    return I, M, vt.shape[2], K


def reconstruct_w_hip(sign, u, vt):
    """(sign * u @ vt).sum(0) from unpacked int8 signs [I, M, N]
    (reconstruct_w_triton, inference_utils.py:135-156)."""
    dev = _lib.require_gpu(sign, u, vt)
    I, M, N, K = _dims(u, vt)
    if tuple(sign.shape) != (I, M, N) or sign.dtype != torch.int8:
        raise ValueError(f"sign must be int8 [{I},{M},{N}], got {sign.dtype} {tuple(sign.shape)}")
    sign, u, vt = sign.contiguous(), _f16c(u), _f16c(vt)
    w = torch.empty((M, N), dtype=torch.float16, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_reconstruct_w_from_sign(_lib.ptr(sign), _lib.ptr(u), _lib.ptr(vt),
                                                         _lib.ptr(w), I, M, N, K, _lib.stream_ptr(dev)),
                   "bs_reconstruct_w_from_sign")
    return w


def unpack_and_reconstruct_w_hip(packed_sign, u, vt):
    """(sign * u @ vt).sum(0) straight from packed signs [I, M*N/8]
    (unpack_and_reconstruct_w_triton and _v2, inference_utils.py:371-387, :465-488)."""
    w = _lib.host().rebuild(packed_sign, u, vt, u.shape[0])
    if w is not None:
        return w
    dev = _lib.require_gpu(packed_sign, u, vt)
    I, M, N, K = _dims(u, vt)
    if packed_sign.dtype != torch.uint8 or packed_sign.numel() != I * ((M * N + 7) // 8):
        raise ValueError(f"packed signs must be uint8 with {I}*{(M * N + 7) // 8} bytes, got "
                         f"{packed_sign.dtype} {tuple(packed_sign.shape)}")
    packed_sign, u, vt = packed_sign.contiguous(), _f16c(u), _f16c(vt)
    w = torch.empty((M, N), dtype=torch.float16, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_reconstruct_w(_lib.ptr(packed_sign), _lib.ptr(u), _lib.ptr(vt),
                                               _lib.ptr(w), I, M, N, K, _lib.stream_ptr(dev)),
                   "bs_reconstruct_w")
    return w


def bitstack_forward_hip(packed_sign, u, vt, x, bias=None):
    """y = x @ (sum_i sign_i * u_i @ vt_i)^T (+ bias) from packed signs; x is
    [..., N] fp16 (reconstruct_and_forward_triton, inference_utils.py:252-284,
    generalised to packed input, any leading shape and an optional bias)."""
    y = _lib.host().forward(packed_sign, u, vt, u.shape[0], x, bias)
    if y is not None:
        return y
    dev = _lib.require_gpu(packed_sign, u, vt, x, bias)
    I, M, N, K = _dims(u, vt)
    if x.shape[-1] != N:
        raise ValueError(f"x has {x.shape[-1]} input features, the layer has {N}")
    if packed_sign.dtype != torch.uint8 or packed_sign.numel() != I * ((M * N + 7) // 8):
        raise ValueError("packed signs do not match u / vt")
    packed_sign, u, vt, x2 = packed_sign.contiguous(), _f16c(u), _f16c(vt), _f16c(x).view(-1, N)
    if bias is not None:
        bias = _f16c(bias)
    T = x2.shape[0]
    y = torch.empty((T, M), dtype=torch.float16, device=dev)
    L = _lib.lib()
    need = L.bs_workspace_bytes(I, M, N, K, T)
    if need < 0:
        _lib.check(int(need), "bs_workspace_bytes")
    with torch.cuda.device(dev), _lib.scratch(dev, need) as ws:
        _lib.check(L.bs_forward(_lib.ptr(packed_sign), _lib.ptr(u), _lib.ptr(vt), _lib.ptr(x2),
                                _lib.ptr(bias), _lib.ptr(y), I, M, N, K, T, _lib.ptr(ws),
                                ws.numel(), _lib.stream_ptr(dev)), "bs_forward")
    return y.view(x.shape[:-1] + (M,))


class MatrixGroup:
    """Up to four stacked BitStack matrices with the same in_features and rank that
    are always applied to the same input (q/k/v, gate/up): the argument block of
    bs_forward_group, built once.  Keeps the tensors alive."""

    def __init__(self, mats):
        # mats: sequence of (packed_sign [I, M*N/8], u [I, M, K], vt [I, K, N], bias or None)
        self.tensors = []
        self.M = []
        arr = (_lib.bs_matrix * len(mats))()
        N = K = None
        for j, (q, u, vt, bias) in enumerate(mats):
            _lib.require_gpu(q, u, vt, bias)
            I, M, n, k = _dims(u, vt)
            if N is None:
                N, K = n, k
            elif (n, k) != (N, K):
                raise ValueError("matrices of a group share in_features and rank")
            if q.dtype != torch.uint8 or q.numel() != I * ((M * n + 7) // 8):
                raise ValueError("packed signs do not match u / vt")
            q, u, vt = q.contiguous(), _f16c(u), _f16c(vt)
            bias = None if bias is None else _f16c(bias)
            self.tensors.append((q, u, vt, bias))
            arr[j].packed, arr[j].u, arr[j].vt = q.data_ptr(), u.data_ptr(), vt.data_ptr()
            arr[j].bias = None if bias is None else bias.data_ptr()
            arr[j].I, arr[j].M = I, M
            self.M.append(M)
        self.arr, self.n, self.N, self.K = arr, len(mats), N, K
        self.dev = mats[0][0].device
        self._need = {}

    @classmethod
    def from_modules(cls, modules):
        """modules: BitStackLinear objects after stack_blocks(), using their first w_bit blocks."""
        mats = []
        for m in modules:
            q, u, vt = m._stacked()
            mats.append((q, u, vt, m.bias))
        return cls(mats)

    def workspace_bytes(self, T, again=False):
        if again or T not in self._need:
            self._need[T] = int(_lib.lib().bs_forward_group_workspace_bytes(self.arr, self.n, self.N, self.K, T))
        return self._need[T]


def bitstack_forward_group_hip(group: MatrixGroup, x, epilogue=_lib.EPI_NONE, residual=None, out=None, rms_eps=None):
    """All matrices of `group` applied to x [T, N] (T <= 48) in one launch, with
    the outputs side by side [T, sum M] (EPI_NONE), plus `residual` (EPI_RESIDUAL),
    or silu(first) * second [T, M] (EPI_SWIGLU).  What three (two) module calls and
    the element-wise ops after them do in a decoder layer.  With rms_eps set, x is
    the un-normalised row and every output is scaled by rsqrt(mean(x^2) + rms_eps)
    (the norm's weight vector must already be folded into the group's vt)."""
    dev = _lib.require_gpu(x, residual, out)
    x2 = _f16c(x).view(-1, group.N)
    T = x2.shape[0]
    width = group.M[0] if epilogue == _lib.EPI_SWIGLU else sum(group.M)
    need = group.workspace_bytes(T)
    if need < 0:
        _lib.check(need, "bs_forward_group_workspace_bytes")
    if residual is not None:
        residual = _f16c(residual)
        if residual.numel() != T * width:
            raise ValueError("residual does not match the output")
    y = out if out is not None else torch.empty((T, width), dtype=torch.float16, device=dev)
    if y.dtype != torch.float16 or not y.is_contiguous() or y.numel() != T * width:
        raise ValueError("out must be a contiguous fp16 [T, width] tensor")
    def call(need):
        with torch.cuda.device(dev), _lib.scratch(dev, need) as ws:
            behind = (_lib.ptr(residual), _lib.ptr(y), _lib.ptr(ws), ws.numel(), _lib.stream_ptr(dev))
            if rms_eps is None:
                return _lib.lib().bs_forward_group(group.arr, group.n, group.N, group.K, _lib.ptr(x2), T, epilogue, *behind)
            return _lib.lib().bs_forward_group_rms(group.arr, group.n, group.N, group.K, _lib.ptr(x2), T, float(rms_eps), epilogue, *behind)

    status = call(need)
    if status == _lib.ERR_WORKSPACE:             # another kernel has been pinned since (bs_set_decode_kernel): its scratch may be larger
        status = call(group.workspace_bytes(T, again=True))
    _lib.check(status, "bs_forward_group" if rms_eps is None else "bs_forward_group_rms")
    return y


def _norm_weight(weight, H):
    if weight.numel() != H:
        raise ValueError(f"a norm of {H} columns needs as many weights, got {tuple(weight.shape)}")
    return _f16c(weight)


def rmsnorm_hip(x, weight, eps, out=None):
    """weight * fp16(x * rsqrt(mean(x^2) + eps)) over the last dimension."""
    dev = _lib.require_gpu(x, weight, out)
    H = x.shape[-1]
    x2, weight = _f16c(x).view(-1, H), _norm_weight(weight, H)
    y = out if out is not None else torch.empty_like(x2)
    if y.dtype != torch.float16 or not y.is_contiguous() or y.numel() != x2.numel():
        raise ValueError("out must be a contiguous fp16 tensor of x's size")
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_rmsnorm_f16(_lib.ptr(x2), _lib.ptr(weight), _lib.ptr(y), x2.shape[0], H, float(eps),
                                             _lib.stream_ptr(dev)), "bs_rmsnorm_f16")
    return y.view(x.shape)


def add_rmsnorm_hip(x, add, weight, eps):
    """(x + add, its RMSNorm): the sum takes the place of `add` (fp16, contiguous) and is returned."""
    dev = _lib.require_gpu(x, add, weight)
    H = x.shape[-1]
    if x.dtype != torch.float16:             # a residual that is kept wider stays so
        x = x + add
        return x, rmsnorm_hip(x, weight, eps)
    if add.dtype != torch.float16 or not add.is_contiguous() or add.shape != x.shape:
        raise ValueError("add must be a contiguous fp16 tensor of x's shape")
    x2, weight = _f16c(x).view(-1, H), _norm_weight(weight, H)
    y = torch.empty_like(x2)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_add_rmsnorm_f16(_lib.ptr(x2), _lib.ptr(add), _lib.ptr(add), _lib.ptr(weight), _lib.ptr(y), x2.shape[0], H,
                                                 float(eps), _lib.stream_ptr(dev)), "bs_add_rmsnorm_f16")
    return add, y.view(x.shape)


def _rows(t, shape):
    """Row stride of a fp16 matrix whose rows are contiguous (a column slice of a wider one, for instance)."""
    if t.dtype != torch.float16 or tuple(t.shape) != tuple(shape) or t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        raise ValueError(f"expected a fp16 matrix {tuple(shape)} with contiguous rows, got {t.dtype} {tuple(t.shape)} {t.stride()}")
    return t.stride(0)


def rope_store_hip(q, k, v, cos, sin, kcache, vcache, n):
    """Positions 0 .. n - 1 of B sequences: RoPE on q [B * n, heads * d] in place, rotated k and v [B * n, kv * d] into the
    caches [B, kv, max_len, d].  q, k and v may be column slices of one wider matrix."""
    dev = _lib.require_gpu(q, k, v, cos, sin, kcache, vcache)
    B, kv, max_len, d = kcache.shape
    for t, shape in ((cos, (max_len, d // 2)), (sin, (max_len, d // 2)), (kcache, kcache.shape), (vcache, kcache.shape)):
        if t.dtype != torch.float16 or not t.is_contiguous() or tuple(t.shape) != tuple(shape):
            raise ValueError(f"expected a contiguous fp16 tensor {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
    if n > max_len or q.shape[1] % d:
        raise ValueError("q must hold whole heads, n at most max_len positions")
    ldq, ldk, ldv = _rows(q, (B * n, q.shape[1])), _rows(k, (B * n, kv * d)), _rows(v, (B * n, kv * d))
    if ldk != ldv:
        raise ValueError("k and v must have the same row stride")
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_rope_store_f16(_lib.ptr(q), ldq, _lib.ptr(k), _lib.ptr(v), ldk, _lib.ptr(cos), _lib.ptr(sin),
                                                _lib.ptr(kcache), _lib.ptr(vcache), B, n, q.shape[1] // d, kv, d, max_len,
                                                _lib.stream_ptr(dev)), "bs_rope_store_f16")


def attention_prefill_hip(q, kcache, vcache, n):
    """Causal attention of positions 0 .. n - 1: q [B * n, heads * 128] rotated (rows may be strided), k and v in the caches
    [B, kv, max_len, 128]; returns [B * n, heads * 128]."""
    dev = _lib.require_gpu(q, kcache, vcache)
    B, kv, max_len, d = kcache.shape
    for t in (kcache, vcache):
        if t.dtype != torch.float16 or not t.is_contiguous():
            raise ValueError("the caches must be contiguous fp16 tensors")
    if vcache.shape != kcache.shape or q.dim() != 2 or q.shape[1] % d or n > max_len:
        raise ValueError("q must hold whole heads of B * n positions, n at most max_len")
    ldq = _rows(q, (B * n, q.shape[1]))
    y = torch.empty(q.shape, dtype=torch.float16, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_attention_prefill_f16(_lib.ptr(q), ldq, _lib.ptr(kcache), _lib.ptr(vcache), _lib.ptr(y), B, n,
                                                       q.shape[1] // d, kv, d, max_len, _lib.stream_ptr(dev)), "bs_attention_prefill_f16")
    return y


def silu_mul_hip(gate, up):
    """silu(gate) * up of two fp16 matrices: in gate's place if both are contiguous, else (column slices) a new matrix."""
    dev = _lib.require_gpu(gate, up)
    if up.shape != gate.shape or up.dtype != torch.float16 or gate.dtype != torch.float16:
        raise ValueError("gate and up must be fp16 tensors of one shape")
    if gate.is_contiguous() and up.is_contiguous():
        y, T, width = gate, 1, gate.numel()
        if width >= 1 << 31:                 # (the kernel counts a row in 32 bits)
            T, width = gate.numel() // gate.shape[-1], gate.shape[-1]
        ld = width
    else:
        T, width = gate.shape
        y, ld = torch.empty(T, width, dtype=torch.float16, device=dev), _rows(gate, gate.shape)
        if _rows(up, gate.shape) != ld:
            raise ValueError("gate and up must have the same row stride")
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_silu_mul_f16(_lib.ptr(gate), _lib.ptr(up), _lib.ptr(y), T, width, ld, _lib.stream_ptr(dev)),
                   "bs_silu_mul_f16")
    return y


def plainly_called(module):
    """Whether a call of `module` is BitStackLinear's own forward and nothing else: no hook, of the module or of all modules, and no
    forward of the instance.  Only then does nobody else see its input or hold its output."""
    from bitstack_amd.modules.BitStackLinear import BitStackLinear
    return (type(module) is BitStackLinear and "forward" not in module.__dict__ and not module._forward_hooks and not module._forward_pre_hooks
            and not module._backward_hooks and not module._backward_pre_hooks and not torch.nn.modules.module._has_any_global_hook())


def forward_cat_hip(modules, x):
    """[T, M0 + M1 + ..]: what the modules (BitStackLinear, level 5) give for x [T, N], side by side from one product, or None
    where that is not how they are computed (few tokens, a bias, another level, blocks not stacked)."""
    args = []
    for m in modules:
        # (a call of the module would do more, or something else)
        if not plainly_called(m) or m.fused_level != 5 or m.no_avd or m.bias is not None:
            return None
        d = m.__dict__
        args += (d.get("qweight"), d.get("u"), d.get("vt"), m.w_bit)
    return _lib.host().forward_cat(x, *args)


def attention_decode_hip(qkv, kcache, vcache, cos, sin, pos, heads, kv_heads, out=None):
    """One decode position for B sequences: RoPE on q and k of qkv [B, (heads + 2 kv) * d],
    append k, v at *pos to the caches [B, kv, max_len, d], attention over 0..*pos;
    returns [B, heads * d].  `pos` is a one-element int64 device tensor."""
    dev = _lib.require_gpu(qkv, kcache, vcache, cos, sin, pos, out)
    B = qkv.shape[0]
    d = kcache.shape[-1]
    max_len = kcache.shape[-2]
    if qkv.dtype != torch.float16 or not qkv.is_contiguous() or qkv.shape[1] != (heads + 2 * kv_heads) * d:
        raise ValueError("qkv must be contiguous fp16 [B, (heads + 2 kv_heads) * head_dim]")
    for c in (kcache, vcache):
        if c.dtype != torch.float16 or not c.is_contiguous() or c.numel() != B * kv_heads * max_len * d:
            raise ValueError("caches must be contiguous fp16 [B, kv_heads, max_len, head_dim]")
    if pos.dtype != torch.int64 or pos.numel() != 1:
        raise ValueError("pos must be a one-element int64 tensor")
    if cos.shape != (max_len, d // 2) or sin.shape != (max_len, d // 2) or not cos.is_contiguous() or not sin.is_contiguous():
        raise ValueError("cos / sin must be contiguous [max_len, head_dim / 2]")
    y = out if out is not None else torch.empty((B, heads * d), dtype=torch.float16, device=dev)
    need = max(0, int(_lib.lib().bs_attention_decode_workspace_bytes(B, heads, kv_heads, d, max_len)))     # (an error is the call's to report)
    with torch.cuda.device(dev), _lib.scratch(dev, need) as ws:
        _lib.check(_lib.lib().bs_attention_decode_ws_f16(_lib.ptr(qkv), _lib.ptr(kcache), _lib.ptr(vcache), _lib.ptr(_f16c(cos)),
                                                         _lib.ptr(_f16c(sin)), _lib.ptr(pos), _lib.ptr(y), B, heads, kv_heads, d, max_len,
                                                         _lib.ptr(ws), ws.numel(), _lib.stream_ptr(dev)),
                   "bs_attention_decode_ws_f16")
    return y


def argmax_hip(x, out=None):
    """Index of the largest value of every row of x [B, V] (fp16), int64 [B]."""
    if out is not None and _lib.host().argmax(x, out):
        return out
    dev = _lib.require_gpu(x, out)
    if x.dim() != 2 or x.dtype != torch.float16 or not x.is_contiguous():
        raise ValueError("x must be a contiguous fp16 [B, V] tensor")
    y = out if out is not None else torch.empty(x.shape[0], dtype=torch.int64, device=dev)
    if y.dtype != torch.int64 or y.numel() != x.shape[0] or not y.is_contiguous():
        raise ValueError("out must be a contiguous int64 [B] tensor")
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_argmax_f16(_lib.ptr(x), _lib.ptr(y), x.shape[0], x.shape[1], _lib.stream_ptr(dev)),
                   "bs_argmax_f16")
    return y


# ---- requests of unequal lengths: a cache in pages -----------------------------------------------------------------------
def _vector(t, n, dtype, name):
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor [{n}], got {t.dtype} {tuple(t.shape)}")


class PagePlan(NamedTuple):
    """What page_plan_hip gives: positions per request and the ring's {first, count} afterwards, tokens that got slots [B], first
    token row of every request [B + 1], position (int32) and slot (int64) of every token row, slot of every request's first token [B];
    -1 without one."""
    lengths: torch.Tensor
    state: torch.Tensor
    granted: torch.Tensor
    starts: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    row_slots: torch.Tensor


def page_plan_hip(lengths, new_tokens, block_table, free_pages, free_state, page_size, tokens, released=None, inplace=False):
    """The pages of a step's tokens, once for all layers.  Request b holds lengths[b] positions and gets new_tokens[b] more (int32 [B]); where
    `released` [B] (bool) is set its pages go back first.  Pages come from the ring free_pages [pool] with free_state = {first, count} (int32 [2]);
    a new pool is free_pages = arange(pool), free_state = [0, pool].  block_table [B, max_pages] and the ring are written in place, lengths and
    free_state too with `inplace` (else new tensors are given back).  `tokens` is the number of token rows, at least sum(new_tokens)."""
    plan = _lib.host().page_plan(lengths, new_tokens, block_table, free_pages, free_state, page_size, tokens, released, bool(inplace))
    if plan is not None:
        return PagePlan._make(plan)
    dev = _lib.require_gpu(lengths, new_tokens, block_table, free_pages, free_state, released)
    B, tokens = lengths.shape[0] if lengths.dim() == 1 else -1, int(tokens)
    _vector(lengths, B, torch.int32, "lengths")
    _vector(new_tokens, B, torch.int32, "new_tokens")
    _vector(free_pages, free_pages.numel(), torch.int32, "free_pages")
    _vector(free_state, 2, torch.int32, "free_state")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B or not block_table.is_contiguous():
        raise ValueError(f"block_table must be a contiguous int32 tensor [{B}, max_pages], got {block_table.dtype} {tuple(block_table.shape)}")
    if released is not None:
        if released.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f"released must be bool or uint8, got {released.dtype}")
        _vector(released, B, released.dtype, "released")
    need = int(_lib.lib().bs_page_plan_workspace_bytes(B, tokens))
    if need < 0:
        _lib.check(need, "bs_page_plan_workspace_bytes")
    i32 = dict(dtype=torch.int32, device=dev)
    plan = PagePlan(lengths if inplace else torch.empty(B, **i32), free_state if inplace else torch.empty(2, **i32), torch.empty(B, **i32),
                    torch.empty(B + 1, **i32), torch.empty(tokens, **i32), torch.empty(tokens, dtype=torch.int64, device=dev),
                    torch.empty(B, dtype=torch.int64, device=dev))
    with torch.cuda.device(dev), _lib.scratch(dev, need, own=True) as ws:
        _lib.check(_lib.lib().bs_page_plan(_lib.ptr(lengths), _lib.ptr(new_tokens), _lib.ptr(released), _lib.ptr(block_table), _lib.ptr(free_pages),
                                           _lib.ptr(free_state), *(_lib.ptr(t) for t in plan), B, tokens, int(page_size), block_table.shape[1],
                                           free_pages.shape[0], _lib.ptr(ws), ws.numel(), _lib.stream_ptr(dev)), "bs_page_plan")
    return plan


def _pages(kpages, vpages, cos, sin):
    """(pool, kv_heads, page_size, head_dim) of a cache in pages, and the positions of the RoPE tables."""
    for t in (kpages, vpages):
        if t.dtype != torch.float16 or t.dim() != 4 or t.shape != kpages.shape or not t.is_contiguous():
            raise ValueError("kpages and vpages must be contiguous fp16 tensors [pool, kv_heads, page_size, head_dim] of one shape")
    for t in (cos, sin):
        if t.dtype != torch.float16 or t.dim() != 2 or t.shape != cos.shape or 2 * t.shape[1] != kpages.shape[3] or not t.is_contiguous():
            raise ValueError("cos and sin must be contiguous fp16 tensors [positions, head_dim / 2] of one shape")
    return (*kpages.shape, cos.shape[0])


def rope_store_paged_hip(q, k, v, cos, sin, kpages, vpages, positions, slots, out=None):
    """RoPE on the token rows of q [T, heads * d] (in place, or into `out`; None: keys and values alone), rotated k and v [T, kv * d] to their
    slots in the pages [pool, kv, page_size, d].  positions (int32) and slots (int64) as page_plan_hip gives them; rows without a
    slot are left as they are.  q, k and v may be column slices of one wider matrix.  Returns the rotated q."""
    if _lib.host().rope_store_paged(q, k, v, cos, sin, kpages, vpages, positions, slots, out):
        return q if out is None else out
    dev = _lib.require_gpu(q, k, v, cos, sin, kpages, vpages, positions, slots, out)
    pool, kv, page, d, max_pos = _pages(kpages, vpages, cos, sin)
    T = k.shape[0]
    _vector(positions, T, torch.int32, "positions")
    _vector(slots, T, torch.int64, "slots")
    if q is not None and (q.dim() != 2 or q.shape[1] % d or q.shape[1] == 0):
        raise ValueError("q must hold whole heads")
    if out is not None and (q is None or out.shape != q.shape):
        raise ValueError("out must be a tensor of q's shape")
    ldk, ldv = _rows(k, (T, kv * d)), _rows(v, (T, kv * d))
    if ldk != ldv:
        raise ValueError("k and v must have the same row stride")
    ldq = 0 if q is None else _rows(q, (T, q.shape[1]))
    ldo = 0 if out is None else _rows(out, q.shape)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_rope_store_paged_f16(_lib.ptr(q), ldq, _lib.ptr(out), ldo, _lib.ptr(k), _lib.ptr(v), ldk, _lib.ptr(cos), _lib.ptr(sin),
                                                      _lib.ptr(positions), _lib.ptr(slots), _lib.ptr(kpages), _lib.ptr(vpages), T,
                                                      0 if q is None else q.shape[1] // d, kv, d, max_pos, page, pool, _lib.stream_ptr(dev)),
                   "bs_rope_store_paged_f16")
    return q if out is None else out


def attention_paged_hip(qkv, kpages, vpages, cos, sin, block_table, lengths, slots, heads, kv_heads, out=None):
    """One new token per request: RoPE on q and k of qkv [B, (heads + 2 kv) * d] at position lengths[b] - 1, k and v to slots[b] of the pages
    [pool, kv, page_size, d], attention over positions 0 .. lengths[b] - 1 by block_table [B, max_pages]; returns [B, heads * d].
    lengths (int32) and slots (int64) are page_plan_hip's lengths and row_slots; a request without a slot is idle and its row zeros.  A score of -inf weighs
    nothing, one of +inf or NaN makes its head's output NaN."""
    y = _lib.host().attention_paged(qkv, kpages, vpages, cos, sin, block_table, lengths, slots, heads, kv_heads, out)
    if y is not None:
        return y if out is None else out
    dev = _lib.require_gpu(qkv, kpages, vpages, cos, sin, block_table, lengths, slots, out)
    pool, kv, page, d, max_pos = _pages(kpages, vpages, cos, sin)
    B = qkv.shape[0]
    if kv != kv_heads:
        raise ValueError(f"the pages hold {kv} heads, not {kv_heads}")
    ldqkv = _rows(qkv, (B, (heads + 2 * kv_heads) * d))
    _vector(lengths, B, torch.int32, "lengths")
    _vector(slots, B, torch.int64, "slots")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B or not block_table.is_contiguous():
        raise ValueError(f"block_table must be a contiguous int32 tensor [{B}, max_pages], got {block_table.dtype} {tuple(block_table.shape)}")
    y = out if out is not None else torch.empty((B, heads * d), dtype=torch.float16, device=dev)
    if y.dtype != torch.float16 or not y.is_contiguous() or y.numel() != B * heads * d:
        raise ValueError("out must be a contiguous fp16 [B, heads * head_dim] tensor")
    need = int(_lib.lib().bs_attention_paged_workspace_bytes(B, heads, kv_heads, d, page, block_table.shape[1]))
    if need < 0:
        _lib.check(need, "bs_attention_paged_workspace_bytes")
    with torch.cuda.device(dev), _lib.scratch(dev, need, own=True) as ws:
        _lib.check(_lib.lib().bs_attention_paged_f16(_lib.ptr(qkv), ldqkv, _lib.ptr(kpages), _lib.ptr(vpages), _lib.ptr(cos), _lib.ptr(sin), _lib.ptr(block_table),
                                                     _lib.ptr(lengths), _lib.ptr(slots), _lib.ptr(y), B, heads, kv_heads, d, max_pos, page,
                                                     block_table.shape[1], pool, _lib.ptr(ws), ws.numel(), _lib.stream_ptr(dev)), "bs_attention_paged_f16")
    return y


def sample_hip(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
    """The next token of every row of logits [B, V] (fp16, rows may be strided), int64 [B], drawn with the given random numbers uniform [B] of [0, 1).
    temperature, top_p, min_p (fp32 [B]) and top_k (int32 [B]) may be None: temperature 1, all tokens.  A temperature of 0 is argmax_hip.
    What stays and how it is drawn: bs_sample_f16 in include/bitstack_hip.h."""
    y = _lib.host().sample(logits, uniform, temperature, top_k, top_p, min_p, out)
    if y is not None:
        return y if out is None else out
    dev = _lib.require_gpu(logits, uniform, temperature, top_k, top_p, min_p, out)
    if logits.dim() != 2:
        raise ValueError("logits must be a fp16 [B, V] tensor")
    B, V = logits.shape
    ld = _rows(logits, (B, V))
    for name, t, dtype in (("uniform", uniform, torch.float32), ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                           ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if t is not None:
            _vector(t, B, dtype, name)
    y = out if out is not None else torch.empty(B, dtype=torch.int64, device=dev)
    _vector(y, B, torch.int64, "out")
    need = int(_lib.lib().bs_sample_workspace_bytes(B, V))
    if need < 0:
        _lib.check(need, "bs_sample_workspace_bytes")
    with torch.cuda.device(dev), _lib.scratch(dev, need, own=True) as ws:
        _lib.check(_lib.lib().bs_sample_f16(_lib.ptr(logits), ld, _lib.ptr(uniform), _lib.ptr(temperature), _lib.ptr(top_k), _lib.ptr(top_p), _lib.ptr(min_p),
                                            _lib.ptr(y), B, V, _lib.ptr(ws), ws.numel(), _lib.stream_ptr(dev)), "bs_sample_f16")
    return y


# ---- drafted tokens: a tree per request; forked rows; settings on logits -----------------------------------------------------
class TreePlan(NamedTuple):
    """What tree_plan_hip gives for every token row: the position that it is rotated by (int32, -1 for rows that are no node), and the
    nodes of its request that it attends to (int64, bit i for node i)."""
    positions: torch.Tensor
    masks: torch.Tensor


class TreeAccept(NamedTuple):
    """What tree_accept_hip gives: positions per request and the ring's {first, count} afterwards, how many nodes were accepted [B], which
    [B, nodes] (-1 behind them), and the token that each request goes on with (int64 [B], -1 without nodes)."""
    lengths: torch.Tensor
    state: torch.Tensor
    accepted: torch.Tensor
    path: torch.Tensor
    token: torch.Tensor


class PageFork(NamedTuple):
    """What page_fork_hip gives: positions per row and the ring's {first, count} afterwards, 1 or 0 for every row (0: no page was there, it stays)."""
    lengths: torch.Tensor
    state: torch.Tensor
    granted: torch.Tensor


def _table(t, B):
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != B or not t.is_contiguous():
        raise ValueError(f"block_table must be a contiguous int32 tensor [{B}, max_pages], got {t.dtype} {tuple(t.shape)}")


def _trees(lengths, granted, starts):
    B = lengths.shape[0] if lengths.dim() == 1 else -1
    _vector(lengths, B, torch.int32, "lengths")
    _vector(granted, B, torch.int32, "granted")
    _vector(starts, B + 1, torch.int32, "starts")
    return B


def _layers(kpages, vpages, pool):
    """(layers, kv_heads, page_size, head_dim) of a cache in pages, of one layer or of all."""
    for t in (kpages, vpages):
        if t.dtype != torch.float16 or t.dim() not in (4, 5) or t.shape != kpages.shape or not t.is_contiguous():
            raise ValueError("kpages and vpages must be contiguous fp16 tensors [layers, pool, kv_heads, page_size, head_dim] (or without layers) of one shape")
    if kpages.shape[-4] != pool:
        raise ValueError(f"free_pages must hold a number for each of the {kpages.shape[-4]} pages, got {pool}")
    return (kpages.shape[0] if kpages.dim() == 5 else 1, *kpages.shape[-3:])


def tree_plan_hip(parents, lengths, granted, starts):
    """Positions and masks of the drafted tokens, once per step.  Request b's tokens are rows starts[b] .. of parents [T] (int32): the first is the one that it goes
    on with, each other names its parent's number among them, a smaller one than its own (-1: none).  lengths, granted, starts: page_plan_hip's for a step of that many tokens
    per request, at most 64."""
    plan = _lib.host().tree_plan(parents, lengths, granted, starts)
    if plan is not None:
        return TreePlan._make(plan)
    dev = _lib.require_gpu(parents, lengths, granted, starts)
    B, T = _trees(lengths, granted, starts), parents.shape[0] if parents.dim() == 1 else -1
    _vector(parents, T, torch.int32, "parents")
    plan = TreePlan(torch.empty(T, dtype=torch.int32, device=dev), torch.empty(T, dtype=torch.int64, device=dev))
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_tree_plan(_lib.ptr(parents), _lib.ptr(lengths), _lib.ptr(granted), _lib.ptr(starts), _lib.ptr(plan.positions), _lib.ptr(plan.masks), B, T,
                                           _lib.stream_ptr(dev)), "bs_tree_plan")
    return plan


def attention_tree_hip(q, kpages, vpages, block_table, lengths, granted, starts, masks, nodes=64, out=None):
    """Attention of drafted tokens: q [T, heads * d] rotated (rows may be strided), their keys and values stored (rope_store_paged_hip with tree_plan_hip's positions does both),
    over the positions that each request held in the pages [pool, kv, page_size, d] and the nodes that masks [T] names.  lengths, granted, starts as in tree_plan_hip;
    `nodes` is the largest number of them that a request has (up to 64; one with more is left out).  Returns [T, heads * d], zeros in rows that are no node; out must not be q's memory."""
    y = _lib.host().attention_tree(q, kpages, vpages, block_table, lengths, granted, starts, masks, nodes, out)
    if y is not None:
        return y if out is None else out
    dev = _lib.require_gpu(q, kpages, vpages, block_table, lengths, granted, starts, masks, out)
    B, nodes = _trees(lengths, granted, starts), int(nodes)
    pool, kv, page, d = kpages.shape if kpages.dim() == 4 else (-1, -1, -1, -1)
    _layers(kpages, vpages, pool)
    _table(block_table, B)
    if q.dim() != 2 or q.shape[1] % d or q.shape[1] == 0:
        raise ValueError("q must hold whole heads")
    T, heads = q.shape[0], q.shape[1] // d
    ldq = _rows(q, (T, heads * d))
    _vector(masks, T, torch.int64, "masks")
    y = out if out is not None else torch.empty((T, heads * d), dtype=torch.float16, device=dev)
    if y.dtype != torch.float16 or not y.is_contiguous() or y.numel() != T * heads * d:
        raise ValueError("out must be a contiguous fp16 [T, heads * head_dim] tensor")
    need = int(_lib.lib().bs_attention_tree_workspace_bytes(B, T, nodes, heads, kv, d, page, block_table.shape[1]))
    if need < 0:
        _lib.check(need, "bs_attention_tree_workspace_bytes")
    with torch.cuda.device(dev), _lib.scratch(dev, need, own=True) as ws:
        _lib.check(_lib.lib().bs_attention_tree_f16(_lib.ptr(q), ldq, _lib.ptr(kpages), _lib.ptr(vpages), _lib.ptr(block_table), _lib.ptr(lengths), _lib.ptr(granted),
                                                    _lib.ptr(starts), _lib.ptr(masks), _lib.ptr(y), B, T, nodes, heads, kv, d, page, block_table.shape[1], pool, _lib.ptr(ws),
                                                    ws.numel(), _lib.stream_ptr(dev)), "bs_attention_tree_f16")
    return y


def tree_accept_hip(tokens, parents, targets, slots, lengths, granted, starts, block_table, free_pages, free_state, kpages, vpages, nodes=64, inplace=False):
    """What the model accepts of drafted trees: from every request's first node on the child whose token (tokens [T], int64) is the target (targets [T], int64: what the
    model gives behind each node) of the node that is reached.  The accepted nodes' keys and values move to the places behind the held positions, in all layers of
    kpages, vpages ([layers, pool, kv, page_size, d], or without layers), and the pages behind them go back to the ring.  slots, lengths, granted, starts and the ring are
    page_plan_hip's, parents and nodes as in tree_plan_hip and attention_tree_hip.  The ring is written in place, lengths and free_state too with `inplace`."""
    done = _lib.host().tree_accept(tokens, parents, targets, slots, lengths, granted, starts, block_table, free_pages, free_state, kpages, vpages, nodes, bool(inplace))
    if done is not None:
        return TreeAccept._make(done)
    dev = _lib.require_gpu(tokens, parents, targets, slots, lengths, granted, starts, block_table, free_pages, free_state, kpages, vpages)
    B, T, nodes = _trees(lengths, granted, starts), parents.shape[0] if parents.dim() == 1 else -1, int(nodes)
    for name, t, dtype in (("tokens", tokens, torch.int64), ("parents", parents, torch.int32), ("targets", targets, torch.int64), ("slots", slots, torch.int64)):
        _vector(t, T, dtype, name)
    _vector(free_pages, free_pages.numel(), torch.int32, "free_pages")
    _vector(free_state, 2, torch.int32, "free_state")
    _table(block_table, B)
    layers, kv, page, d = _layers(kpages, vpages, free_pages.shape[0])
    if not 1 <= nodes <= 64:
        raise ValueError("nodes must be 1 to 64")
    need = int(_lib.lib().bs_tree_accept_workspace_bytes(B))
    if need < 0:
        _lib.check(need, "bs_tree_accept_workspace_bytes")
    i32 = dict(dtype=torch.int32, device=dev)
    done = TreeAccept(lengths if inplace else torch.empty(B, **i32), free_state if inplace else torch.empty(2, **i32), torch.empty(B, **i32), torch.empty(B, nodes, **i32),
                      torch.empty(B, dtype=torch.int64, device=dev))
    with torch.cuda.device(dev), _lib.scratch(dev, need, own=True) as ws:
        _lib.check(_lib.lib().bs_tree_accept_f16(*(_lib.ptr(t) for t in (tokens, parents, targets, slots, lengths, granted, starts, block_table, free_pages, free_state, kpages,
                                                                         vpages, *done)), B, T, nodes, layers, kv, d, page, block_table.shape[1], free_pages.shape[0],
                                                 _lib.ptr(ws), ws.numel(), _lib.stream_ptr(dev)), "bs_tree_accept_f16")
    return done


def page_fork_hip(source, lengths, block_table, free_pages, free_state, shares, kpages, vpages, inplace=False):
    """Rows of a paged cache become copies of other rows: row b what row source[b] (int32 [B]) was, -1 empty, its own number the row that it is.  Whole pages are shared
    (shares [pool], int32, zeros in a new pool: holders less one), a last page that is not full is copied in all layers of kpages, vpages ([layers, pool, kv, page_size, d], or
    without layers) to a new one; pages that nobody holds any more go back to the ring.  Rows that share pages must not be released by page_plan_hip.
    block_table, the ring and shares are written in place, lengths and free_state too with `inplace`."""
    done = _lib.host().page_fork(source, lengths, block_table, free_pages, free_state, shares, kpages, vpages, bool(inplace))
    if done is not None:
        return PageFork._make(done)
    dev = _lib.require_gpu(source, lengths, block_table, free_pages, free_state, shares, kpages, vpages)
    B = lengths.shape[0] if lengths.dim() == 1 else -1
    _vector(lengths, B, torch.int32, "lengths")
    _vector(source, B, torch.int32, "source")
    _vector(free_pages, free_pages.numel(), torch.int32, "free_pages")
    _vector(shares, free_pages.numel(), torch.int32, "shares")
    _vector(free_state, 2, torch.int32, "free_state")
    _table(block_table, B)
    layers, kv, page, d = _layers(kpages, vpages, free_pages.shape[0])
    need = int(_lib.lib().bs_page_fork_workspace_bytes(B, block_table.shape[1], free_pages.shape[0]))
    if need < 0:
        _lib.check(need, "bs_page_fork_workspace_bytes")
    i32 = dict(dtype=torch.int32, device=dev)
    done = PageFork(lengths if inplace else torch.empty(B, **i32), free_state if inplace else torch.empty(2, **i32), torch.empty(B, **i32))
    with torch.cuda.device(dev), _lib.scratch(dev, need, own=True) as ws:
        _lib.check(_lib.lib().bs_page_fork_f16(*(_lib.ptr(t) for t in (source, lengths, block_table, free_pages, free_state, shares, kpages, vpages, *done)), B, layers, kv, d,
                                               page, block_table.shape[1], free_pages.shape[0], _lib.ptr(ws), ws.numel(), _lib.stream_ptr(dev)), "bs_page_fork_f16")
    return done


def _given(t, shape, dtype, name):
    """A contiguous tensor of that type and shape (None: any size), or None."""
    if t is not None and (t.dtype != dtype or t.dim() != len(shape) or any(want is not None and want != got for want, got in zip(shape, t.shape)) or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {list(shape)}, got {t.dtype} {tuple(t.shape)}")


def logits_adjust_hip(logits, history=None, history_lengths=None, prompt_lengths=None, repetition=None, frequency=None, presence=None, drafted=None, requests=None,
                      bias_tokens=None, bias=None, allowed=None, allowed_rows=None, out=None):
    """Penalties, biases and grammar masks on logits [R, V] (fp16, rows may be strided), in place or into `out`; returns what was written.  Row r belongs to request requests[r]
    (int32; None: r).  history [B, n] (int32) are the requests' tokens, history_lengths and prompt_lengths [B] how many of them there are and belong to the prompt, drafted [R, m]
    more tokens of single rows (-1: none); repetition, frequency and presence [B] (fp32) are the penalties.  bias [B, k] (fp32) is added for bias_tokens [B, k] (int32, -1:
    none).  allowed [masks, ceil(V / 32)] (int32) has a bit for each token, allowed_rows [R] (int32; None: r) says which mask a row uses (-1: none).  What is computed, in
    which order: bs_logits_adjust_f16 in include/bitstack_hip.h."""
    y = _lib.host().logits_adjust(logits, history, history_lengths, prompt_lengths, repetition, frequency, presence, drafted, requests, bias_tokens, bias, allowed, allowed_rows,
                                  out)
    if y:
        return logits if out is None else out
    dev = _lib.require_gpu(logits, history, history_lengths, prompt_lengths, repetition, frequency, presence, drafted, requests, bias_tokens, bias, allowed, allowed_rows, out)
    if logits.dim() != 2:
        raise ValueError("logits must be a fp16 [R, V] tensor")
    R, V = logits.shape
    ld = _rows(logits, (R, V))
    y = logits if out is None else out
    ldo = _rows(y, (R, V))
    if (history is None and (history_lengths is not None or prompt_lengths is not None)) or (bias is None) != (bias_tokens is None) or (allowed is None and allowed_rows is not None):
        raise ValueError("history_lengths and prompt_lengths go with history, bias with bias_tokens, allowed_rows with allowed")
    if history is None and drafted is None and any(t is not None for t in (repetition, frequency, presence)):
        raise ValueError("penalties need history or drafted tokens")
    per_request = [t.shape[0] for t in (history, history_lengths, prompt_lengths, repetition, frequency, presence, bias_tokens, bias) if t is not None]
    B = per_request[0] if per_request else R
    i32, f32 = torch.int32, torch.float32
    for t, shape, dtype, name in ((history, (B, None), i32, "history"), (history_lengths, (B,), i32, "history_lengths"), (prompt_lengths, (B,), i32, "prompt_lengths"),
                                  (repetition, (B,), f32, "repetition"), (frequency, (B,), f32, "frequency"), (presence, (B,), f32, "presence"),
                                  (drafted, (R, None), i32, "drafted"), (requests, (R,), i32, "requests"), (bias_tokens, (B, None), i32, "bias_tokens"),
                                  (bias, (B, None), f32, "bias"), (allowed, (None, (V + 31) // 32), i32, "allowed"), (allowed_rows, (R,), i32, "allowed_rows")):
        _given(t, shape, dtype, name)
    if bias is not None and bias.shape != bias_tokens.shape:
        raise ValueError("bias must have the shape of bias_tokens")
    if (requests is None and B != R) or (allowed is not None and allowed_rows is None and allowed.shape[0] != R):
        raise ValueError(f"without requests and allowed_rows there must be one request and one mask for each of the {R} rows")
    width = lambda t: 0 if t is None else t.shape[1]                       # noqa: E731
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_logits_adjust_f16(_lib.ptr(logits), ld, _lib.ptr(y), ldo, _lib.ptr(requests), _lib.ptr(history), width(history), _lib.ptr(history_lengths),
                                                   _lib.ptr(prompt_lengths), _lib.ptr(repetition), _lib.ptr(frequency), _lib.ptr(presence), _lib.ptr(drafted), width(drafted),
                                                   _lib.ptr(bias_tokens), _lib.ptr(bias), width(bias), _lib.ptr(allowed), 0 if allowed is None else allowed.shape[0],
                                                   _lib.ptr(allowed_rows), R, V, B, _lib.stream_ptr(dev)), "bs_logits_adjust_f16")
    return y


def linear_f16_hip(x, w, bias=None):
    """F.linear on the library's own MFMA kernel (fp16 in, fp32 accumulate)."""
    y = _lib.host().linear(x, w, bias)
    if y is not None:
        return y
    dev = _lib.require_gpu(x, w, bias)
    M, N = w.shape
    x2, w = _f16c(x).view(-1, N), _f16c(w)
    if bias is not None:
        bias = _f16c(bias)
    T = x2.shape[0]
    y = torch.empty((T, M), dtype=torch.float16, device=dev)
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().bs_linear_f16(_lib.ptr(x2), _lib.ptr(w), _lib.ptr(bias), _lib.ptr(y),
                                            T, M, N, _lib.stream_ptr(dev)), "bs_linear_f16")
    return y.view(x.shape[:-1] + (M,))


def reconstruct_and_forward_hip(sign, u, vt, x):
    """Reference signature of level 5 (unpacked int8 signs, 3-D x, no bias;
    inference_utils.py:252-284): rebuild the weight, then the MFMA linear."""
    if x.dim() != 3:
        raise ValueError("x must be [BZ, L, N]")
    return linear_f16_hip(x, reconstruct_w_hip(sign, u, vt))


# drop-in aliases for code written against the reference's names
reconstruct_w_triton = reconstruct_w_hip
unpack_and_reconstruct_w_triton = unpack_and_reconstruct_w_hip
unpack_and_reconstruct_w_triton_v2 = unpack_and_reconstruct_w_hip
unpack_and_reconstruct_w_triton_v3 = unpack_and_reconstruct_w_hip
reconstruct_and_forward_triton = reconstruct_and_forward_hip
