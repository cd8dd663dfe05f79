"""A mixture-of-experts layer for a few tokens, over the C ABI (b200_moe_layer)."""
from __future__ import annotations

from . import api
from .api import STATUS_WORKSPACE, GemmError
from .mx import FORMATS, MxTensor, _current, _elsewhere, _half_type, _invalid, _output, _require_cuda, _Torch

torch = _Torch(globals())

MAX_TOKENS, MAX_EXPERTS, MAX_TOP_K, MAX_SIZE = 64, 512, 32, 2 ** 20


def moe_workspace_bytes(tokens: int, experts: int, top_k: int, hidden: int, inner: int) -> int:
    """Bytes of ``workspace`` for these sizes; 0 for sizes that moe_layer does not take."""
    if max(abs(n) for n in (tokens, experts, top_k, hidden, inner)) > MAX_SIZE:
        return 0  # (the C ABI takes 32-bit numbers)
    return int(api.library().b200_moe_workspace_bytes(tokens, experts, top_k, hidden, inner))


def _workspace_bytes(tokens: int, top_k: int, inner: int) -> int:
    """b200_moe_workspace_bytes of sizes that are known to be within the limits."""
    pairs = tokens * top_k
    return (pairs * inner * 4 + 255) // 256 * 256 + (pairs * 4 + 255) // 256 * 512


def moe_layer(x, router, w_gate_up, w_down, top_k: int, bias=None, renormalize: bool = True, out=None,
              return_routing: bool = False, workspace=None, stream=None):
    """out[T, H] = sum over each token's top_k experts e of p[t, e] * W2[e] (silu(G[e] x[t]) * (U[e] x[t])).

    ``x`` [T, H] (at most 64 tokens), ``router`` [E, H], ``bias`` [E] fp32 added to the router's logits (-inf
    takes an expert out), ``w_gate_up`` [E, 2 I, H] (the gate's I rows, then the up projection's),
    ``w_down`` [E, H, I]: bfloat16 or float16, one type. Or, with bfloat16 tokens, 4-bit experts: ``w_gate_up`` an
    MxTensor of E * 2 I rows and H columns, ``w_down`` one of E * H rows and I columns. ``renormalize``: the
    softmax runs over the chosen experts, otherwise over all of them.

    With ``return_routing`` the result is ``(out, ids, weights)``: the chosen experts [T, top_k] (int32, largest
    logit first, -1 where fewer experts than top_k are left) and their weights (fp32). A token without any
    expert gets zeros. No history for gradients is recorded. Expert weights have to be finite. With float16 a hidden value beyond 65504 is infinite.
    include/b200_gemm.h has the rounding and the limits.
    """
    f16 = _half_type(x.dtype, "x")
    if x.dim() != 2 or router.dim() != 2 or router.shape[1] != x.shape[1]:
        raise _invalid("x must be [tokens, hidden] and router [experts, hidden]")
    T, H = x.shape
    E = router.shape[0]
    if not 1 <= T <= MAX_TOKENS:
        raise _invalid(f"1 to {MAX_TOKENS} tokens, got {T}")
    if not 1 <= E <= MAX_EXPERTS or not 1 <= top_k <= min(E, MAX_TOP_K):
        raise _invalid(f"1 to {MAX_EXPERTS} experts and a top_k of 1 to {MAX_TOP_K}, at most all experts")
    four_bit = isinstance(w_gate_up, MxTensor)
    if four_bit != isinstance(w_down, MxTensor):
        raise _invalid("w_gate_up and w_down must both be 4-bit or both not")
    if four_bit:
        if f16:
            raise _invalid("4-bit experts take bfloat16 tokens")
        if w_gate_up.format != w_down.format:
            raise _invalid(f"w_gate_up is {w_gate_up.format}, w_down is {w_down.format}")
        I = w_down.cols
        if w_gate_up.cols != H or w_gate_up.rows != E * 2 * I or w_down.rows != E * H:
            raise _invalid(f"w_gate_up must be a [{E} * 2 I, {H}] and w_down a [{E} * {H}, I] matrix")
    else:
        if w_gate_up.dim() != 3 or w_down.dim() != 3:
            raise _invalid("w_gate_up must be [experts, 2 I, hidden] and w_down [experts, hidden, I]")
        I = w_down.shape[2]
        if w_gate_up.shape != (E, 2 * I, H) or w_down.shape != (E, H, I):
            raise _invalid(f"w_gate_up must be [{E}, 2 I, {H}] and w_down [{E}, {H}, I]")
    if H % 8 or I % 8 or H == 0 or I == 0:
        raise _invalid("hidden and inner sizes must be multiples of 8")
    if H > MAX_SIZE or I > MAX_SIZE:
        raise _invalid(f"hidden and inner sizes of at most {MAX_SIZE}, got {H} and {I}")
    device, dtype = x.device, x.dtype
    _require_cuda(device, "x")

    def pointer(t, name, dtype, align=16):
        if t.device != device:
            _require_cuda(t.device, name, device)
        if t.dtype is not dtype or not t.is_contiguous():
            raise _invalid(f"{name} must be a contiguous {dtype} tensor")
        p = t.data_ptr()
        if p % align:
            raise _invalid(f"{name} must start on {align} bytes")
        return p

    x_ptr, router_ptr = pointer(x, "x", dtype), pointer(router, "router", dtype)
    bias_ptr = None
    if bias is not None:
        if bias.shape != (E,):
            raise _invalid(f"bias must have shape ({E},)")
        bias_ptr = pointer(bias, "bias", torch.float32, 4)
    if out is not None:
        _output(out, (T, H), dtype, device, True)
    need = _workspace_bytes(T, top_k, I)
    if workspace is not None:
        _require_cuda(workspace.device, "workspace", device)
        if workspace.numel() * workspace.element_size() < need or not workspace.is_contiguous():
            raise GemmError(STATUS_WORKSPACE, f"workspace needs {need} contiguous bytes")
    if four_bit:
        _require_cuda(w_gate_up.device, "w_gate_up", device)
        _require_cuda(w_down.device, "w_down", device)
        w1 = (FORMATS[w_gate_up.format], w_gate_up._data_ptr, w_gate_up._scales_ptr, w_gate_up.tensor_scale)
        w2 = (w_down._data_ptr, w_down._scales_ptr, w_down.tensor_scale)
    else:
        w1 = (-1, pointer(w_gate_up, "w_gate_up", dtype), None, 1.0)
        w2 = (pointer(w_down, "w_down", dtype), None, 1.0)

    sizes = (f16, T, E, top_k, H, I, x_ptr, router_ptr, bias_ptr, *w1, *w2, 1 if renormalize else 0)
    handle = _current(device, stream)
    if handle is not False:
        return _launch(x, sizes, need, top_k, out, return_routing, workspace, handle)
    with _elsewhere(device, stream) as handle:
        return _launch(x, sizes, need, top_k, out, return_routing, workspace, handle)


def _launch(x, sizes, need, top_k, out, return_routing, workspace, handle):
    device = x.device
    if out is None:
        out = torch.empty_like(x)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    ids = weights = ids_ptr = weights_ptr = None
    if return_routing:
        ids = torch.empty(x.shape[0], top_k, dtype=torch.int32, device=device)
        weights = torch.empty(x.shape[0], top_k, dtype=torch.float32, device=device)
        ids_ptr, weights_ptr = ids.data_ptr(), weights.data_ptr()
    rc = api.library().b200_moe_layer(*sizes, out.data_ptr(), ids_ptr, weights_ptr, workspace.data_ptr(), need, handle)
    if rc:
        api._check(rc)
    return (out, ids, weights) if return_routing else out
