"""Torch-facing wrappers of the C ABI (device memory and streams come from torch).

Every function validates dtype, device and contiguity the way the reference's
Python layer does, allocates outputs and workspace with the torch caching
allocator, enqueues on the current CUDA stream and raises ``RuntimeError``
with the library's status text on failure.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Sequence

import torch

from moeinfra_b200 import _native
from moeinfra_b200._native import NF4Expert, NF4Matrix, check

NF4_BLOCKSIZE = 64
NESTED_BLOCKSIZE = 256


def _p(t: torch.Tensor | None) -> ctypes.c_void_p | None:
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _on_device(fn):
    """Run a wrapper with the device of its first CUDA tensor (or device) argument current.

    The library launches on the stream it is given, and CUDA requires that stream to belong
    to the current device (torch's default stream is the null handle: the current device's
    own).  A call on another GPU's tensors than the current one switches devices for its
    duration, and only then."""
    @functools.wraps(fn)
    def wrapper(*args, **kwargs):
        dev = None
        for a in (*args, *kwargs.values()):
            if isinstance(a, torch.Tensor) and a.is_cuda:
                dev = a.device.index
                break
            if isinstance(a, torch.device) and a.type == "cuda" and a.index is not None:
                dev = a.index
                break
        if dev is None or dev == torch.cuda.current_device():
            return fn(*args, **kwargs)
        with torch.cuda.device(dev):
            return fn(*args, **kwargs)
    return wrapper


def _need_cuda(what: str, **tensors: torch.Tensor) -> torch.device:
    dev = None
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a torch.Tensor")
        if t.device.type != "cuda":
            raise RuntimeError(
                f"{what}: {name} is on {t.device}; the B200 kernels run on CUDA tensors only "
                "(there is no CPU path)")
        if not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{what}: {name} is on {t.device}, expected {dev}")
    assert dev is not None
    return dev


def _need_dtype(what: str, t: torch.Tensor, dtype: torch.dtype, name: str) -> None:
    if t.dtype != dtype:
        raise ValueError(f"{what}: {name} must be {dtype}, got {t.dtype}")


# Rows an expert stage call may have on the decode kernels (MOE_DECODE_MAX_ROWS).
DECODE_MAX_ROWS = 8


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)


def check_device(device: torch.device | int | None = None) -> None:
    """Synchronise the current stream of ``device`` and raise if a kernel flagged an error.

    Kernels never trap: a bounded wait that ran out, or experts of one launch
    with different codebooks, leave a bit in the device error word and the
    launch's outputs invalid.  Call this where the caller synchronises anyway
    (the end of a step, before reading results back).
    """
    dev = torch.device("cuda", torch.cuda.current_device() if device is None else
                       (device if isinstance(device, int) else device.index))
    with torch.cuda.device(dev):
        status = _native.stream_check(torch.cuda.current_stream(dev).cuda_stream)
    if status != 0:
        raise RuntimeError(f"device check failed: {_native.status_string(status)} (status {status})")


@_on_device
def probe_wait(flag: torch.Tensor, target: int = 1) -> torch.Tensor:
    """One bounded device wait until ``flag[0] >= target``; returns the device-side wait time (ns)."""
    dev = _need_cuda("probe_wait", flag=flag)
    _need_dtype("probe_wait", flag, torch.int32, "flag")
    waited = torch.zeros(1, dtype=torch.int32, device=dev)
    check(_native.lib().moe_probe_wait(_p(flag), int(target), _p(waited), _stream(dev)),
          "moe_probe_wait")
    return waited


# ---------------------------------------------------------------------------
# NF4 dequant
# ---------------------------------------------------------------------------

@_on_device
def nf4_dequant(q: torch.Tensor, absmax: torch.Tensor, code: torch.Tensor, numel: int,
                blocksize: int = NF4_BLOCKSIZE) -> torch.Tensor:
    """bf16 ``code[nib(i)] * absmax[i // blocksize]`` (bit-exact), flat [numel]."""
    dev = _need_cuda("nf4_dequant", q=q, absmax=absmax, code=code)
    _need_dtype("nf4_dequant", q, torch.uint8, "q")
    _need_dtype("nf4_dequant", absmax, torch.float32, "absmax")
    _need_dtype("nf4_dequant", code, torch.float32, "code")
    if q.numel() * 2 < numel or absmax.numel() * blocksize < numel or code.numel() < 16:
        raise ValueError("nf4_dequant: buffers too small for numel")
    out = torch.empty(numel, dtype=torch.bfloat16, device=dev)
    check(_native.lib().moe_nf4_dequant(_p(q), _p(absmax), _p(code), numel, blocksize, _p(out),
                                        _stream(dev)), "moe_nf4_dequant")
    return out


@_on_device
def nf4_tile16(q: torch.Tensor, absmax: torch.Tensor, rows: int, cols: int):
    """Store layout -> tile16 device layout (exact permutation); returns (q_t, absmax_t)."""
    dev = _need_cuda("nf4_tile16", q=q, absmax=absmax)
    _need_dtype("nf4_tile16", q, torch.uint8, "q")
    _need_dtype("nf4_tile16", absmax, torch.float32, "absmax")
    if q.numel() * 2 != rows * cols or absmax.numel() * NF4_BLOCKSIZE != rows * cols:
        raise ValueError("nf4_tile16: tensor sizes do not match rows x cols")
    q_out = torch.empty_like(q.reshape(-1))
    a_out = torch.empty_like(absmax.reshape(-1))
    check(_native.lib().moe_nf4_tile16(_p(q), _p(absmax), rows, cols, _p(q_out), _p(a_out),
                                       _stream(dev)), "moe_nf4_tile16")
    return q_out, a_out


@_on_device
def nf4_dequant_tile16(q: torch.Tensor, absmax: torch.Tensor, code: torch.Tensor, rows: int,
                       cols: int) -> torch.Tensor:
    """bf16 [rows, cols] of a tile16 matrix (bit-exact with the store-layout dequant)."""
    dev = _need_cuda("nf4_dequant_tile16", q=q, absmax=absmax, code=code)
    out = torch.empty(rows, cols, dtype=torch.bfloat16, device=dev)
    check(_native.lib().moe_nf4_dequant_tile16(_p(q), _p(absmax), _p(code), rows, cols, _p(out),
                                               _stream(dev)), "moe_nf4_dequant_tile16")
    return out


@_on_device
def nested_absmax(qabs: torch.Tensor, absmax2: torch.Tensor, code2: torch.Tensor,
                  offset: float, blocksize2: int = NESTED_BLOCKSIZE) -> torch.Tensor:
    dev = _need_cuda("nested_absmax", qabs=qabs, absmax2=absmax2, code2=code2)
    _need_dtype("nested_absmax", qabs, torch.uint8, "qabs")
    _need_dtype("nested_absmax", absmax2, torch.float32, "absmax2")
    _need_dtype("nested_absmax", code2, torch.float32, "code2")
    n = qabs.numel()
    if absmax2.numel() * blocksize2 < n or code2.numel() < 256:
        raise ValueError("nested_absmax: nested state too small")
    out = torch.empty(n, dtype=torch.float32, device=dev)
    check(_native.lib().moe_nf4_nested_absmax(_p(qabs), _p(absmax2), _p(code2), float(offset), n,
                                              blocksize2, _p(out), _stream(dev)),
          "moe_nf4_nested_absmax")
    return out


# ---------------------------------------------------------------------------
# Router
# ---------------------------------------------------------------------------

@_on_device
def router_topk(h: torch.Tensor, wg: torch.Tensor, k: int, with_logits: bool = True):
    """``(logits fp16 [T,E] | None, weights fp32 [T,k], indices int64 [T,k])``."""
    dev = _need_cuda("router_topk", h=h, wg=wg)
    _need_dtype("router_topk", h, torch.float16, "hidden_states")
    _need_dtype("router_topk", wg, torch.float16, "gate_weight")
    T, H = h.shape
    E = wg.shape[0]
    logits = torch.empty(T, E, dtype=torch.float16, device=dev) if with_logits else None
    w = torch.empty(T, k, dtype=torch.float32, device=dev)
    idx = torch.empty(T, k, dtype=torch.int64, device=dev)
    check(_native.lib().moe_router_topk(_p(h), _p(wg), T, H, E, k, _p(logits), _p(w), _p(idx),
                                        _stream(dev)), "moe_router_topk")
    return logits, w, idx


@_on_device
def router_topk_from_logits(logits: torch.Tensor, k: int):
    dev = _need_cuda("router_topk_from_logits", logits=logits)
    _need_dtype("router_topk_from_logits", logits, torch.float16, "logits")
    T, E = logits.shape
    w = torch.empty(T, k, dtype=torch.float32, device=dev)
    idx = torch.empty(T, k, dtype=torch.int64, device=dev)
    check(_native.lib().moe_router_topk_from_logits(_p(logits), T, E, k, _p(w), _p(idx),
                                                    _stream(dev)), "moe_router_topk_from_logits")
    return w, idx


# ---------------------------------------------------------------------------
# Experts and the fused layer
# ---------------------------------------------------------------------------

def matrix_desc(q: torch.Tensor, absmax: torch.Tensor, code: torch.Tensor) -> NF4Matrix:
    return NF4Matrix(q.data_ptr(), absmax.data_ptr(), code.data_ptr())


@_on_device
def expert_forward(desc: NF4Expert, x: torch.Tensor, hidden: int, inter: int) -> torch.Tensor:
    dev = _need_cuda("expert_forward", x=x)
    _need_dtype("expert_forward", x, torch.float16, "x")
    if x.ndim != 2 or x.shape[1] != hidden:
        raise ValueError(f"expert_forward: x must be [n, {hidden}], got {tuple(x.shape)}")
    n = x.shape[0]
    y = torch.empty(n, hidden, dtype=torch.float16, device=dev)
    lib = _native.lib()
    ws_bytes = lib.moe_expert_workspace_size(n, hidden, inter)
    ws = _workspace(ws_bytes, dev)
    check(lib.moe_expert_forward(ctypes.byref(desc), _p(x), n, hidden, inter, _p(y), _p(ws),
                                 ws_bytes, _stream(dev)), "moe_expert_forward")
    return y


def expert_array(descs: Sequence[NF4Expert]):
    arr = (NF4Expert * len(descs))()
    for i, d in enumerate(descs):
        arr[i] = d
    return arr


# Decode-sized layer calls reuse one workspace (and routing scratch) per
# (device, stream, shape): calls on one stream are ordered, and every kernel
# of the layer waits for its predecessor before it touches the workspace.
_DECODE_WS_MAX_TOKENS = 8
_layer_ws: dict = {}


def _layer_scratch(dev: torch.device, stream: int, T: int, hidden: int, inter: int, E: int, k: int):
    key = (dev.index, stream, T, hidden, inter, E, k)
    ent = _layer_ws.get(key)
    if ent is None:
        ws_bytes = _native.lib().moe_layer_workspace_size(T, hidden, inter, E, k)
        ent = (_workspace(ws_bytes, dev), ws_bytes,
               torch.empty(T, k, dtype=torch.int64, device=dev),
               torch.empty(T, k, dtype=torch.float32, device=dev))
        if T <= _DECODE_WS_MAX_TOKENS:
            _layer_ws[key] = ent
    return ent


@_on_device
def layer_forward(h: torch.Tensor, wg: torch.Tensor, experts, k: int, hidden: int, inter: int,
                  out: torch.Tensor | None = None, routing: bool = True):
    """Fused MoE layer: returns ``(out fp16 [T,H], indices int64 [T,k], weights fp32 [T,k])``.

    ``experts`` is a ctypes array of ``NF4Expert`` (see :func:`expert_array`).
    ``routing=False``: the caller discards indices and weights (returned as
    None; the kernels write them to reused scratch).
    """
    dev = _need_cuda("layer_forward", h=h, wg=wg)
    _need_dtype("layer_forward", h, torch.float16, "hidden_states")
    _need_dtype("layer_forward", wg, torch.float16, "gate_weight")
    T = h.shape[0]
    E = len(experts)
    if out is None:
        out = torch.empty(T, hidden, dtype=torch.float16, device=dev)
    stream = torch.cuda.current_stream(dev).cuda_stream
    ws, ws_bytes, idx, w = _layer_scratch(dev, stream, T, hidden, inter, E, k)
    if routing:
        idx = torch.empty(T, k, dtype=torch.int64, device=dev)
        w = torch.empty(T, k, dtype=torch.float32, device=dev)
    check(_native.lib().moe_layer_forward(_p(h), _p(wg), experts, E, k, T, hidden, inter, _p(out),
                                          _p(idx), _p(w), _p(ws), ws_bytes,
                                          ctypes.c_void_p(stream)), "moe_layer_forward")
    return (out, idx, w) if routing else (out, None, None)


@_on_device
def layer_forward_noalloc(h: torch.Tensor, wg: torch.Tensor, experts, k: int, hidden: int,
                          inter: int, out: torch.Tensor | None = None):
    """:func:`layer_forward` with the library's own static device scratch (no workspace).

    At most ``MOE_NOALLOC_SCRATCH_BYTES`` of scratch; calls overlapping on one
    device must be serialised.
    """
    dev = _need_cuda("layer_forward_noalloc", h=h, wg=wg)
    _need_dtype("layer_forward_noalloc", h, torch.float16, "hidden_states")
    _need_dtype("layer_forward_noalloc", wg, torch.float16, "gate_weight")
    T = h.shape[0]
    if out is None:
        out = torch.empty(T, hidden, dtype=torch.float16, device=dev)
    idx = torch.empty(T, k, dtype=torch.int64, device=dev)
    w = torch.empty(T, k, dtype=torch.float32, device=dev)
    # The library takes the scratch of the CURRENT device: make it h's.
    with torch.cuda.device(dev):
        check(_native.lib().moe_layer_forward_noalloc(_p(h), _p(wg), experts, len(experts), k, T,
                                                      hidden, inter, _p(out), _p(idx), _p(w),
                                                      _stream(dev)), "moe_layer_forward_noalloc")
    return out, idx, w


@_on_device
def routed_layer_forward(h: torch.Tensor, indices: torch.Tensor, weights: torch.Tensor, experts,
                         hidden: int, inter: int) -> torch.Tensor:
    """The MoE layer on routing the caller already has (indices int64 / weights fp32 [T, k]).

    permute -> gather -> experts -> ordered fp16 combine, with no second
    routing pass; every expert slot without tokens in ``indices`` is never read.
    """
    E = len(experts)
    offsets, pair_token, _, pair_slot = permute(indices.contiguous(), weights.contiguous(), E)
    x_sorted = gather_rows(h.contiguous(), pair_token)
    y_sorted = experts_forward(experts, offsets, x_sorted, hidden, inter)
    return combine(y_sorted, pair_slot, indices.contiguous(), weights.contiguous())


@_on_device
def experts_forward(experts, expert_offsets: torch.Tensor, x_sorted: torch.Tensor, hidden: int,
                    inter: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """Expert stage on rows grouped by expert (``expert_offsets`` int32 [E+1] on device)."""
    dev = _need_cuda("experts_forward", expert_offsets=expert_offsets, x_sorted=x_sorted)
    _need_dtype("experts_forward", x_sorted, torch.float16, "x_sorted")
    _need_dtype("experts_forward", expert_offsets, torch.int32, "expert_offsets")
    P = x_sorted.shape[0]
    if out is None:
        out = torch.empty(P, hidden, dtype=torch.float16, device=dev)
    lib = _native.lib()
    ws_bytes = lib.moe_experts_workspace_size(P, hidden, inter)
    ws = _workspace(ws_bytes, dev)
    check(lib.moe_experts_forward(experts, len(experts), _p(expert_offsets), _p(x_sorted), P,
                                  hidden, inter, _p(out), _p(ws), ws_bytes, _stream(dev)),
          "moe_experts_forward")
    return out


@_on_device
def permute(indices: torch.Tensor, weights: torch.Tensor, num_experts: int):
    dev = _need_cuda("permute", indices=indices, weights=weights)
    _need_dtype("permute", indices, torch.int64, "indices")
    _need_dtype("permute", weights, torch.float32, "weights")
    T, k = indices.shape
    P = T * k
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    pair_token = torch.empty(P, dtype=torch.int32, device=dev)
    pair_weight = torch.empty(P, dtype=torch.float32, device=dev)
    pair_slot = torch.empty(P, dtype=torch.int32, device=dev)
    check(_native.lib().moe_permute(_p(indices), _p(weights), T, k, num_experts, _p(offsets),
                                    _p(pair_token), _p(pair_weight), _p(pair_slot), _stream(dev)),
          "moe_permute")
    return offsets, pair_token, pair_weight, pair_slot


@_on_device
def gather_rows(rows: torch.Tensor, index: torch.Tensor) -> torch.Tensor:
    dev = _need_cuda("gather_rows", rows=rows, index=index)
    _need_dtype("gather_rows", rows, torch.float16, "rows")
    _need_dtype("gather_rows", index, torch.int32, "index")
    out = torch.empty(index.numel(), rows.shape[1], dtype=torch.float16, device=dev)
    check(_native.lib().moe_gather_rows(_p(rows), _p(index), index.numel(), rows.shape[1], _p(out),
                                        _stream(dev)), "moe_gather_rows")
    return out


@_on_device
def combine(y_sorted: torch.Tensor, pair_slot: torch.Tensor, indices: torch.Tensor,
            weights: torch.Tensor) -> torch.Tensor:
    dev = _need_cuda("combine", y_sorted=y_sorted, pair_slot=pair_slot, indices=indices,
                     weights=weights)
    _need_dtype("combine", y_sorted, torch.float16, "y_sorted")
    T, k = indices.shape
    width = y_sorted.shape[1]
    out = torch.empty(T, width, dtype=torch.float16, device=dev)
    check(_native.lib().moe_combine(_p(y_sorted), _p(pair_slot), _p(indices), _p(weights), T, k,
                                    width, _p(out), _stream(dev)), "moe_combine")
    return out


# ---------------------------------------------------------------------------
# Expert-parallel exchange (pack / receive / return around two all-to-alls)
# ---------------------------------------------------------------------------

@_on_device
def ep_dispatch(h: torch.Tensor, offsets: torch.Tensor, pair_token: torch.Tensor,
                pair_slot: torch.Tensor, k: int, num_experts: int, world: int, cap: int):
    """``(send_rows fp16 [world*(cap+1), H], pair_slot_ep int32 [T*k])``.

    Chunk r of ``send_rows`` is cap token rows for rank r followed by a header
    row holding rank r's expert counts (int32).
    """
    dev = _need_cuda("ep_dispatch", h=h, offsets=offsets)
    _need_dtype("ep_dispatch", h, torch.float16, "hidden_states")
    T, H = h.shape
    send = torch.empty(world * (cap + 1), H, dtype=torch.float16, device=dev)
    slot_ep = torch.empty(T * k, dtype=torch.int32, device=dev)
    check(_native.lib().moe_ep_dispatch(_p(h), _p(offsets), _p(pair_token), _p(pair_slot), T, k,
                                        num_experts, world, cap, H, _p(send), None,
                                        _p(slot_ep), _stream(dev)), "moe_ep_dispatch")
    return send, slot_ep


@_on_device
def ep_receive(recv_rows: torch.Tensor, num_experts: int, world: int, cap: int):
    """``(x_sorted fp16 [world*cap, H], local_offsets int32 [E/world + 1], recv_counts int32 [E])``."""
    dev = _need_cuda("ep_receive", recv_rows=recv_rows)
    H = recv_rows.shape[1]
    x = torch.empty(world * cap, H, dtype=torch.float16, device=dev)
    off = torch.empty(num_experts // world + 1, dtype=torch.int32, device=dev)
    counts = torch.empty(num_experts, dtype=torch.int32, device=dev)
    check(_native.lib().moe_ep_receive(_p(recv_rows), _p(counts), num_experts, world, cap, H,
                                       _p(x), _p(off), _stream(dev)), "moe_ep_receive")
    return x, off, counts


@_on_device
def ep_return(y_sorted: torch.Tensor, recv_counts: torch.Tensor, num_experts: int, world: int,
              cap: int) -> torch.Tensor:
    """``y_back fp16 [world*cap, H]`` in the exchanged (source rank, row) layout."""
    dev = _need_cuda("ep_return", y_sorted=y_sorted, recv_counts=recv_counts)
    H = y_sorted.shape[1]
    y_back = torch.empty(world * cap, H, dtype=torch.float16, device=dev)
    check(_native.lib().moe_ep_return(_p(y_sorted), _p(recv_counts), num_experts, world, cap, H,
                                      _p(y_back), _stream(dev)), "moe_ep_return")
    return y_back


# ---------------------------------------------------------------------------
# Expert-parallel exchange over peer memory (see moeinfra_b200.ep_p2p)
# ---------------------------------------------------------------------------

@_on_device
def ep_dispatch_p2p(h: torch.Tensor, offsets: torch.Tensor, pair_token: torch.Tensor,
                    pair_slot: torch.Tensor, k: int, num_experts: int, world: int, rank: int,
                    cap: int, peer_recv: int, peer_flags: int, seq: int, done: int) -> torch.Tensor:
    """Rows straight into the owners' receive regions, then signal; returns pair_slot_ep."""
    dev = _need_cuda("ep_dispatch_p2p", h=h, offsets=offsets)
    T, H = h.shape
    slot_ep = torch.empty(T * k, dtype=torch.int32, device=dev)
    check(_native.lib().moe_ep_dispatch_p2p(_p(h), _p(offsets), _p(pair_token), _p(pair_slot), T,
                                            k, num_experts, world, rank, cap, H,
                                            ctypes.c_void_p(peer_recv), ctypes.c_void_p(peer_flags),
                                            ctypes.c_void_p(seq), ctypes.c_void_p(done),
                                            _p(slot_ep), _stream(dev)), "moe_ep_dispatch_p2p")
    return slot_ep


@_on_device
def ep_return_p2p(y_sorted: torch.Tensor, recv_counts: torch.Tensor, num_experts: int, world: int,
                  rank: int, cap: int, peer_back: int, peer_flags: int, seq: int, done: int) -> None:
    dev = _need_cuda("ep_return_p2p", y_sorted=y_sorted, recv_counts=recv_counts)
    check(_native.lib().moe_ep_return_p2p(_p(y_sorted), _p(recv_counts), num_experts, world, rank,
                                          cap, y_sorted.shape[1], ctypes.c_void_p(peer_back),
                                          ctypes.c_void_p(peer_flags), ctypes.c_void_p(seq),
                                          ctypes.c_void_p(done), _stream(dev)), "moe_ep_return_p2p")


@_on_device
def ep_wait_p2p(flags: int, world: int, seq: int, device: torch.device) -> None:
    check(_native.lib().moe_ep_wait_p2p(ctypes.c_void_p(flags), world, ctypes.c_void_p(seq),
                                        _stream(device)), "moe_ep_wait_p2p")


@_on_device
def ep_receive_rows(recv_rows: torch.Tensor, num_experts: int, world: int, cap: int):
    """:func:`ep_receive` on a receive region that is a view (peer-memory exchange)."""
    return ep_receive(recv_rows, num_experts, world, cap)


@_on_device
def ep_receive_p2p(recv_rows: torch.Tensor, num_experts: int, world: int, cap: int, flags: int,
                   seq: int):
    """:func:`ep_receive` of a peer-memory receive region, waiting (bounded, in the kernel)
    for all ``world`` flags at ``flags`` to reach ``*seq`` first."""
    dev = _need_cuda("ep_receive_p2p", recv_rows=recv_rows)
    H = recv_rows.shape[1]
    x = torch.empty(world * cap, H, dtype=torch.float16, device=dev)
    off = torch.empty(num_experts // world + 1, dtype=torch.int32, device=dev)
    counts = torch.empty(num_experts, dtype=torch.int32, device=dev)
    check(_native.lib().moe_ep_receive_p2p(_p(recv_rows), _p(counts), num_experts, world, cap, H,
                                           _p(x), _p(off), ctypes.c_void_p(flags),
                                           ctypes.c_void_p(seq), _stream(dev)),
          "moe_ep_receive_p2p")
    return x, off, counts


@_on_device
def combine_p2p(y_back: torch.Tensor, pair_slot: torch.Tensor, indices: torch.Tensor,
                weights: torch.Tensor, world: int, flags: int, seq: int) -> torch.Tensor:
    """:func:`combine` of a peer-memory return region, waiting (bounded, in the kernel) for all
    ``world`` flags at ``flags`` to reach ``*seq`` first."""
    dev = _need_cuda("combine_p2p", y_back=y_back, pair_slot=pair_slot, indices=indices,
                     weights=weights)
    _need_dtype("combine_p2p", y_back, torch.float16, "y_back")
    T, k = indices.shape
    width = y_back.shape[1]
    out = torch.empty(T, width, dtype=torch.float16, device=dev)
    check(_native.lib().moe_combine_p2p(_p(y_back), _p(pair_slot), _p(indices), _p(weights), T,
                                        k, width, _p(out), ctypes.c_void_p(flags), world,
                                        ctypes.c_void_p(seq), _stream(dev)), "moe_combine_p2p")
    return out


@_on_device
def ep_front_p2p(h: torch.Tensor, gate_f16: torch.Tensor, k: int, num_experts: int, world: int,
                 rank: int, cap: int, peer_recv: int, peer_flags: int, seq: int, done: int,
                 bar: int, zero: torch.Tensor | None = None):
    """Router, permute and the peer-memory dispatch in one launch (``T`` <= the SM count).

    Returns ``(weights fp32 [T, k], indices int64 [T, k], pair_slot_ep int32 [T*k])``, the
    values :func:`router_topk`, :func:`permute` and :func:`ep_dispatch_p2p` give.  ``zero``
    (int32, optional) is zeroed by the same launch: the counters of the expert stage that
    follows (:func:`experts_forward_partials` ``counters``)."""
    dev = _need_cuda("ep_front_p2p", h=h, gate_f16=gate_f16)
    _need_dtype("ep_front_p2p", h, torch.float16, "h")
    _need_dtype("ep_front_p2p", gate_f16, torch.float16, "gate_f16")
    T, H = h.shape
    w = torch.empty(T, k, dtype=torch.float32, device=dev)
    idx = torch.empty(T, k, dtype=torch.int64, device=dev)
    slot_ep = torch.empty(T * k, dtype=torch.int32, device=dev)
    check(_native.lib().moe_ep_front_p2p(_p(h), _p(gate_f16), T, num_experts, k, world, rank, cap,
                                         H, ctypes.c_void_p(peer_recv),
                                         ctypes.c_void_p(peer_flags), ctypes.c_void_p(seq),
                                         ctypes.c_void_p(done), ctypes.c_void_p(bar), _p(w),
                                         _p(idx), _p(slot_ep),
                                         None if zero is None else _p(zero),
                                         0 if zero is None else zero.numel(), _stream(dev)),
          "moe_ep_front_p2p")
    return w, idx, slot_ep


def expert_splits(inter: int) -> int:
    """K splits of the decode down projection (its fp32 partials per row)."""
    return int(_native.lib().moe_expert_splits(inter))


def expert_counter_words(inter: int) -> int:
    """int32 completion counters of the decode expert stage (zeroed before each call)."""
    return int(_native.lib().moe_experts_counter_words(inter))


@_on_device
def experts_forward_partials(experts, expert_offsets: torch.Tensor, x_sorted: torch.Tensor,
                             hidden: int, inter: int,
                             counters: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`experts_forward` of a decode batch (<= 8 rows) up to the down projection's
    fp32 split partials ``[P, S, hidden]`` (their in-order fp16 sum is the output row).
    ``counters``: :func:`expert_counter_words` int32 already zeroed on the stream (by
    :func:`ep_front_p2p`), which spares the zeroing launch; None zeroes internal ones."""
    dev = _need_cuda("experts_forward_partials", expert_offsets=expert_offsets, x_sorted=x_sorted)
    _need_dtype("experts_forward_partials", x_sorted, torch.float16, "x_sorted")
    _need_dtype("experts_forward_partials", expert_offsets, torch.int32, "expert_offsets")
    P = x_sorted.shape[0]
    part = torch.empty(P, expert_splits(inter), hidden, dtype=torch.float32, device=dev)
    lib = _native.lib()
    ws_bytes = lib.moe_experts_workspace_size(P, hidden, inter)
    ws = _workspace(ws_bytes, dev)
    if counters is not None and counters.numel() < expert_counter_words(inter):
        raise ValueError("counters smaller than expert_counter_words(inter)")
    check(lib.moe_experts_forward_partials(experts, len(experts), _p(expert_offsets),
                                           _p(x_sorted), P, hidden, inter, _p(part),
                                           None if counters is None else _p(counters), _p(ws),
                                           ws_bytes, _stream(dev)),
          "moe_experts_forward_partials")
    return part


@_on_device
def ep_return_partials_p2p(y_part: torch.Tensor, recv_counts: torch.Tensor, num_experts: int,
                           world: int, rank: int, cap: int, peer_back: int, peer_flags: int,
                           seq: int, done: int) -> None:
    """:func:`ep_return_p2p` from :func:`experts_forward_partials`' fp32 partials."""
    dev = _need_cuda("ep_return_partials_p2p", y_part=y_part, recv_counts=recv_counts)
    _need_dtype("ep_return_partials_p2p", y_part, torch.float32, "y_part")
    check(_native.lib().moe_ep_return_partials_p2p(
        _p(y_part), y_part.shape[1], _p(recv_counts), num_experts, world, rank, cap,
        y_part.shape[2], ctypes.c_void_p(peer_back), ctypes.c_void_p(peer_flags),
        ctypes.c_void_p(seq), ctypes.c_void_p(done), _stream(dev)), "moe_ep_return_partials_p2p")


# ---------------------------------------------------------------------------
# Ragged, paged serving: rotation + cache append, attention, sampling
#
# A call on one new token is a few microseconds on the GPU, so the wrappers check the usual form
# (packed tensors of one device) in one expression and go through the detailed checks, which
# name what is wrong or accept strided rows, only where that fails.
# ---------------------------------------------------------------------------

_DTYPE_CODES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
PROMPT_WORKSPACE_BYTES = 16
_COUNTER_BYTES = 4096  # the part of a workspace that has to be zero before its first call
_serve_ws: dict = {}
_raw_stream = torch._C._cuda_getCurrentRawStream
_HALVES = (torch.float16, torch.bfloat16)


def _plain(dev: int, dtype: torch.dtype, *tensors) -> bool:
    """Whether all are packed tensors of one type on GPU ``dev``."""
    for t in tensors:
        if t.dtype is not dtype or t.get_device() != dev or not t.is_contiguous():
            return False
    return dev >= 0


def _on_first_device(fn):
    """As :func:`_on_device`, by the device of the first parameter alone."""
    name = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def wrapper(*args, **kwargs):
        first = args[0] if args else kwargs.get(name)
        dev = first.get_device() if isinstance(first, torch.Tensor) else -1
        if dev < 0 or dev == torch.cuda.current_device():
            return fn(*args, **kwargs)
        with torch.cuda.device(dev):
            return fn(*args, **kwargs)
    return wrapper


def _serve_scratch(dev: int, stream: int, nbytes: int) -> torch.Tensor:
    """Scratch of the serving operators, its leading counters zeroed (every call leaves them so).

    One buffer per (device, stream, power of two), kept: calls on one stream are ordered and
    every kernel waits for its predecessor before it touches scratch.  A call under stream
    capture gets scratch of its own, zeroed by the graph: graphs captured on one stream may be
    replayed side by side.
    """
    if torch.cuda.is_current_stream_capturing():
        ws = _workspace(max(nbytes, _COUNTER_BYTES), torch.device("cuda", dev))
        ws[:_COUNTER_BYTES].zero_()
        return ws
    key = (dev, stream, max(nbytes - 1, _COUNTER_BYTES - 1).bit_length())
    ws = _serve_ws.get(key)
    if ws is None:
        ws = _serve_ws[key] = torch.zeros(1 << key[2], dtype=torch.uint8,
                                          device=torch.device("cuda", dev))
    return ws


def _serve_check(what: str, dev: int, *named) -> None:
    """Each of ``named`` = (name, tensor, dtype, shape, packed): dtype and shape as given (None: any
    size), the last ``packed`` dimensions contiguous, on GPU ``dev``."""
    for name, t, dtype, shape, packed in named:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{what}: {name} must be a torch.Tensor")
        if not t.is_cuda:
            raise RuntimeError(
                f"{what}: {name} is on {t.device}; the B200 kernels run on CUDA tensors only "
                "(there is no CPU path)")
        if t.get_device() != dev:
            raise ValueError(f"{what}: {name} is on {t.device}, expected cuda:{dev}")
        if t.dtype is not dtype:
            raise ValueError(f"{what}: {name} must be {dtype}, got {t.dtype}")
        size = t.shape
        if len(size) != len(shape) or any(w is not None and w != n for w, n in zip(shape, size)):
            want = ", ".join("*" if w is None else str(w) for w in shape)
            raise ValueError(f"{what}: {name} must be [{want}], got {tuple(size)}")
        run, stride = 1, t.stride()
        for i in range(len(size) - 1, len(size) - 1 - packed, -1):
            if size[i] != 1 and stride[i] != run:
                raise ValueError(f"{what}: {name} must be contiguous in its last {packed} "
                                 "dimension(s)")
            run *= size[i]


def _check_workspace(what: str, ws: torch.Tensor, dev: int, nbytes: int) -> None:
    """A caller's own workspace: packed, on GPU ``dev``, of ``nbytes`` at least."""
    if not isinstance(ws, torch.Tensor):
        raise TypeError(f"{what}: workspace must be a torch.Tensor")
    if ws.get_device() != dev or not ws.is_contiguous():
        raise ValueError(f"{what}: workspace must be packed and on cuda:{dev}, got {ws.device} "
                         f"with strides {tuple(ws.stride())}")
    if ws.numel() * ws.element_size() < nbytes:
        raise ValueError(f"{what}: workspace needs {nbytes} bytes")


def _outer_stride(t: torch.Tensor) -> int:
    """Elements from one index of the first dimension to the next (packed when there is one)."""
    return t.stride(0) if t.shape[0] > 1 else t.numel()


def _row_strides(t: torch.Tensor) -> tuple[int, int]:
    """Strides of [rows, heads, hd] in elements (packed where a dimension has one entry)."""
    row, head, _ = t.stride()
    if t.shape[1] <= 1:
        head = t.shape[2]
    if t.shape[0] <= 1:
        row = max(t.shape[1], 1) * head
    return row, head


def _check_cache(what: str, k_pages, v_pages, block_table) -> None:
    if not isinstance(k_pages, torch.Tensor) or k_pages.ndim != 4:
        raise ValueError(f"{what}: k_pages must be [pages, kv_heads, page_size, head_dim]")
    if k_pages.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"{what}: k_pages must be float16 or bfloat16, got {k_pages.dtype}")
    dev, dt, shape = k_pages.get_device(), k_pages.dtype, k_pages.shape
    _serve_check(what, dev, ("k_pages", k_pages, dt, shape, 3), ("v_pages", v_pages, dt, shape, 3),
                 ("block_table", block_table, torch.int32, (None, None), 1))
    if shape[3] not in (64, 128):
        raise ValueError(f"{what}: head_dim must be 64 or 128, got {shape[3]}")


@_on_first_device
def rope_append(qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor,
                block_table: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                num_heads: int, seq_ids: torch.Tensor | None = None,
                out: torch.Tensor | None = None, k_out: torch.Tensor | None = None,
                slots: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q and k of fused projection rows and append k and v to the paged cache.

    ``qkv`` [tokens, (num_heads + 2 * kv_heads) * head_dim] (rows may be strided), fp16 or bf16;
    ``cos`` / ``sin`` fp32 [max_positions, head_dim / 2]; ``positions`` int32 [tokens] in the
    token's own sequence (negative: padding, a zero q row and nothing appended); ``block_table``
    int32 [sequences, max_pages]; ``k_pages`` / ``v_pages`` [pages, kv_heads, page_size, head_dim],
    written in place; ``seq_ids`` int32 [tokens] (None: token t is sequence t, the decode step).
    Returns q [tokens, num_heads, head_dim]; ``k_out`` [tokens, kv_heads, head_dim], if given,
    receives the rotated keys packed, as :func:`prompt_attention` reads them.  ``slots`` int32
    [tokens]: where in its sequence a token's keys and values go, if not to its position: drafted
    nodes are rotated by their depth and stored by their index (:func:`tree_attention`).  A
    position, slot, sequence or page out of range appends nothing and shows in :func:`check_device`.
    """
    what = "rope_append"
    try:
        n_pages, kv, page, hd = k_pages.shape
        T, width = qkv.shape
        max_pos, half = cos.shape
        seqs, max_pages = block_table.shape
        dt, dev = k_pages.dtype, k_pages.get_device()
        plain = (dt in _HALVES and (hd == 64 or hd == 128) and half * 2 == hd
                 and width == (num_heads + 2 * kv) * hd and sin.shape == cos.shape
                 and v_pages.shape == k_pages.shape and positions.shape == (T,)
                 and _plain(dev, dt, qkv, k_pages, v_pages)
                 and _plain(dev, torch.float32, cos, sin)
                 and _plain(dev, torch.int32, positions, block_table)
                 and (seq_ids is None or seq_ids.shape == (T,) and _plain(dev, torch.int32, seq_ids)))
    except (AttributeError, ValueError):
        plain = False
    if not plain:
        _check_cache(what, k_pages, v_pages, block_table)
        n_pages, kv, page, hd = k_pages.shape
        dt, dev = k_pages.dtype, k_pages.get_device()
        _serve_check(what, dev, ("qkv", qkv, dt, (None, (num_heads + 2 * kv) * hd), 1),
                     ("cos", cos, torch.float32, (None, hd // 2), 2))
        T, max_pos = qkv.shape[0], cos.shape[0]
        _serve_check(what, dev, ("positions", positions, torch.int32, (T,), 1),
                     ("sin", sin, torch.float32, cos.shape, 2))
        if seq_ids is not None:
            _serve_check(what, dev, ("seq_ids", seq_ids, torch.int32, (T,), 1))
        seqs, max_pages = block_table.shape
    if seq_ids is None and seqs < T:
        raise ValueError(f"{what}: block_table has {seqs} sequences for {T} tokens")
    if out is None:
        out = qkv.new_empty((T, num_heads, hd))
    else:
        _serve_check(what, dev, ("out", out, dt, (T, num_heads, hd), 3))
    if k_out is not None:
        _serve_check(what, dev, ("k_out", k_out, dt, (T, kv, hd), 3))
    if slots is not None:
        _serve_check(what, dev, ("slots", slots, torch.int32, (T,), 1))
    page_elems = kv * page * hd
    strides = ((page_elems, page_elems, max_pages, (num_heads + 2 * kv) * hd) if plain else
               (_outer_stride(k_pages), _outer_stride(v_pages),
                _outer_stride(block_table) if seqs else max_pages,
                _outer_stride(qkv) if T else qkv.shape[1]))
    args = _native.ROPE_APPEND.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), strides[0], strides[1], n_pages, kv, page, hd,
        _DTYPE_CODES[dt], block_table.data_ptr(), strides[2], seqs, max_pages, qkv.data_ptr(),
        strides[3], cos.data_ptr(), sin.data_ptr(), max_pos,
        positions.data_ptr(), 0 if seq_ids is None else seq_ids.data_ptr(), T, num_heads,
        out.data_ptr(), 0 if k_out is None else k_out.data_ptr(), _raw_stream(dev))
    status = (_native.lib().moe_rope_append(args) if slots is None else
              _native.lib().moe_rope_append_slots(args, slots.data_ptr()))
    if status:
        check(status, "moe_rope_append")
    return out


@functools.lru_cache(maxsize=1024)
def _paged_ws_bytes(device: int, seqs: int, max_pages: int, page: int, heads: int, kv: int,
                    hd: int) -> int:
    return _native.lib().moe_paged_attention_workspace_size(seqs, max_pages, page, heads, kv, hd)


@_on_first_device
def paged_attention_workspace(block_table: torch.Tensor, page_size: int, num_heads: int,
                              kv_heads: int, head_dim: int) -> torch.Tensor:
    """A workspace for :func:`paged_attention` calls with these heads, over tables of any size."""
    nbytes = _paged_ws_bytes(block_table.get_device(), *block_table.shape, page_size, num_heads,
                             kv_heads, head_dim)
    return torch.zeros(nbytes, dtype=torch.uint8, device=block_table.device)


@_on_first_device
def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    block_table: torch.Tensor, lengths: torch.Tensor,
                    scale: float | None = None, out: torch.Tensor | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one new token per sequence over its cached keys and values.

    ``q`` [sequences, heads, head_dim] (rows may be strided), ``lengths`` int32 [sequences]: the
    positions each sequence sees, the token just appended included (0: a row of zeros); the rest
    as in :func:`rope_append`; ``page_size`` a multiple of 16.  ``scale`` defaults to
    ``head_dim ** -0.5``.  Returns [sequences, heads, head_dim].

    ``workspace``: a buffer from :func:`paged_attention_workspace` that no call on another
    stream uses at the same time; by default the module keeps one per stream (and a captured
    call zeroes one of its own at every replay, which a given workspace spares).
    """
    what = "paged_attention"
    try:
        n_pages, kv, page, hd = k_pages.shape
        seqs, max_pages = block_table.shape
        rows, heads, _ = q.shape
        dt, dev = k_pages.dtype, k_pages.get_device()
        plain = (dt in _HALVES and (hd == 64 or hd == 128) and q.shape == (seqs, heads, hd)
                 and v_pages.shape == k_pages.shape and lengths.shape == (seqs,)
                 and _plain(dev, dt, q, k_pages, v_pages)
                 and _plain(dev, torch.int32, lengths, block_table))
    except (AttributeError, ValueError):
        plain = False
    if not plain:
        _check_cache(what, k_pages, v_pages, block_table)
        n_pages, kv, page, hd = k_pages.shape
        dt, dev = k_pages.dtype, k_pages.get_device()
        seqs, max_pages = block_table.shape
        _serve_check(what, dev, ("q", q, dt, (seqs, None, hd), 2),
                     ("lengths", lengths, torch.int32, (seqs,), 1))
        heads = q.shape[1]
    if page % 16:
        raise ValueError(f"{what}: page_size must be a multiple of 16, got {page}")
    if heads == 0 or kv == 0 or heads % kv:
        raise ValueError(f"{what}: {heads} query heads do not divide over {kv} KV heads")
    if out is None:
        out = q.new_empty((seqs, heads, hd))
    else:
        _serve_check(what, dev, ("out", out, dt, (seqs, heads, hd), 3))
    if seqs == 0:
        return out
    stream = _raw_stream(dev)
    nbytes = _paged_ws_bytes(dev, seqs, max_pages, page, heads, kv, hd)
    if workspace is None:
        workspace = _serve_scratch(dev, stream, nbytes)
    else:
        _check_workspace(what, workspace, dev, nbytes)
    page_elems = kv * page * hd
    strides = ((page_elems, page_elems, max_pages, heads * hd) if plain else
               (_outer_stride(k_pages), _outer_stride(v_pages), _outer_stride(block_table),
                _outer_stride(q)))
    status = _native.lib().moe_paged_attention(_native.PAGED_ATTENTION.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), strides[0], strides[1], n_pages, kv, page, hd,
        _DTYPE_CODES[dt], block_table.data_ptr(), strides[2], seqs, max_pages, q.data_ptr(),
        strides[3], heads,
        lengths.data_ptr(), hd ** -0.5 if scale is None else scale, out.data_ptr(),
        workspace.data_ptr(), nbytes, stream))
    if status:
        check(status, "moe_paged_attention")
    return out


@_on_first_device
def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     max_seqlen: int, cu_seqlens_k: torch.Tensor | None = None,
                     max_seqlen_k: int | None = None, causal: bool = True,
                     scale: float | None = None, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention over packed prompts of different lengths.

    ``q`` [rows, heads, head_dim], ``k`` / ``v`` [rows_k, kv_heads, head_dim] (rows and heads may
    be strided), fp16 or bf16, head_dim 64 or 128; sequence b's queries are rows
    ``cu_seqlens[b] .. cu_seqlens[b+1]`` (int32, on the device), none longer than ``max_seqlen``;
    its keys likewise by ``cu_seqlens_k`` / ``max_seqlen_k`` (default: the queries').  Causal: the
    queries are the last of their sequence's positions; one that sees no key gives zeros.  Returns
    [rows, heads, head_dim]; rows that belong to no sequence are not written.  ``workspace``: as for :func:`paged_attention`, of at least
    ``PROMPT_WORKSPACE_BYTES`` zeroed bytes (the same buffer may serve both).
    """
    what = "prompt_attention"
    try:
        T, heads, hd = q.shape
        dt, dev = q.dtype, q.get_device()
        plain = (dt in _HALVES and (hd == 64 or hd == 128) and dev >= 0 and k.shape == v.shape
                 and k.ndim == 3 and k.shape[2] == hd and k.dtype is dt and v.dtype is dt
                 and k.get_device() == dev and v.get_device() == dev and cu_seqlens.ndim == 1
                 and q.stride(2) == 1 and k.stride(2) == 1 and v.stride(2) == 1
                 and _plain(dev, torch.int32, cu_seqlens))
    except (AttributeError, ValueError):
        plain = False
    if not plain:
        if not isinstance(q, torch.Tensor) or q.ndim != 3:
            raise ValueError(f"{what}: q must be [rows, heads, head_dim]")
        dt, dev = q.dtype, q.get_device()
        if dt not in _HALVES:
            raise ValueError(f"{what}: q must be float16 or bfloat16, got {dt}")
        T, heads, hd = q.shape
        if hd not in (64, 128):
            raise ValueError(f"{what}: head_dim must be 64 or 128, got {hd}")
        _serve_check(what, dev, ("q", q, dt, q.shape, 1), ("k", k, dt, (None, None, hd), 1))
        _serve_check(what, dev, ("v", v, dt, k.shape, 1),
                     ("cu_seqlens", cu_seqlens, torch.int32, (None,), 1))
    kv, seqs = k.shape[1], cu_seqlens.shape[0] - 1
    if seqs < 0 or kv == 0 or heads == 0 or heads % kv:
        raise ValueError(f"{what}: {heads} query heads do not divide over {kv} KV heads, or "
                         "cu_seqlens is empty")
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens
        if max_seqlen_k is None:
            max_seqlen_k = max_seqlen
    elif max_seqlen_k is None:
        raise ValueError(f"{what}: cu_seqlens_k needs max_seqlen_k")
    else:
        _serve_check(what, dev, ("cu_seqlens_k", cu_seqlens_k, torch.int32, (seqs + 1,), 1))
    if out is None:
        out = q.new_empty((T, heads, hd))
    else:
        _serve_check(what, dev, ("out", out, dt, (T, heads, hd), 3))
    stream = _raw_stream(dev)
    if workspace is None:
        workspace = _serve_scratch(dev, stream, PROMPT_WORKSPACE_BYTES)
    else:
        _check_workspace(what, workspace, dev, PROMPT_WORKSPACE_BYTES)
    status = _native.lib().moe_prompt_attention(_native.PROMPT_ATTENTION.pack(
        q.data_ptr(), *_row_strides(q), T, k.data_ptr(), *_row_strides(k), v.data_ptr(),
        *_row_strides(v), k.shape[0], cu_seqlens.data_ptr(), cu_seqlens_k.data_ptr(), seqs,
        max_seqlen, max_seqlen_k, heads, kv, hd, bool(causal), _DTYPE_CODES[dt],
        hd ** -0.5 if scale is None else scale, out.data_ptr(), workspace.data_ptr(),
        PROMPT_WORKSPACE_BYTES, stream))
    if status:
        check(status, "moe_prompt_attention")
    return out


@_on_first_device
def sample_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperature: torch.Tensor,
                  top_k: torch.Tensor, top_p: torch.Tensor, min_p: torch.Tensor):
    """``(tokens int64 [rows], probs fp32 [rows])``: one token per row of ``logits`` [rows, vocab].

    ``logits`` fp16, bf16 or fp32 (rows may be strided, or one row expanded; vocab <= 262144); ``uniforms`` fp32 [rows]
    in [0, 1), the row's random number; ``temperature`` / ``top_p`` / ``min_p`` fp32 and ``top_k``
    int32 [rows].  Temperature 0 takes the maximum (lowest index); top_k 0, top_p 1 and min_p 0 are
    off; the filters apply in that order, top-p to what top-k leaves.  ``probs`` is the token's
    share of what the filters leave.  The same row and numbers give the same token in any batch.
    """
    what = "sample_tokens"
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2:
        raise ValueError(f"{what}: logits must be [rows, vocab]")
    code = _DTYPE_CODES.get(logits.dtype)
    if code is None:
        raise ValueError(f"{what}: logits must be float16, bfloat16 or float32, got {logits.dtype}")
    dev = logits.get_device()
    rows, vocab = logits.shape
    f32 = torch.float32
    per_row = (rows,)
    try:
        plain = (uniforms.shape == per_row and temperature.shape == per_row
                 and top_k.shape == per_row and top_p.shape == per_row and min_p.shape == per_row
                 and _plain(dev, f32, uniforms, temperature, top_p, min_p)
                 and _plain(dev, torch.int32, top_k) and (logits.stride(1) == 1 or vocab == 1))
    except AttributeError:
        plain = False
    if not plain:
        _serve_check(what, dev, ("logits", logits, logits.dtype, logits.shape, 1),
                     ("uniforms", uniforms, f32, per_row, 1),
                     ("temperature", temperature, f32, per_row, 1),
                     ("top_k", top_k, torch.int32, per_row, 1),
                     ("top_p", top_p, f32, per_row, 1), ("min_p", min_p, f32, per_row, 1))
    tokens = logits.new_empty(rows, dtype=torch.int64)
    probs = logits.new_empty(rows, dtype=f32)
    status = _native.lib().moe_sample_tokens(_native.SAMPLE_TOKENS.pack(
        logits.data_ptr(), _outer_stride(logits), rows, vocab, code, uniforms.data_ptr(),
        temperature.data_ptr(), top_k.data_ptr(), top_p.data_ptr(), min_p.data_ptr(),
        tokens.data_ptr(), probs.data_ptr(), _raw_stream(dev)))
    if status:
        check(status, "moe_sample_tokens")
    return tokens, probs


# ---------------------------------------------------------------------------
# Several continuations of a sequence over the paged cache: trees of drafted tokens, beams
# ---------------------------------------------------------------------------


def _check_layers(what: str, k_pages, v_pages, block_table) -> tuple:
    """The cache's shape and strides as ``FORK_PAGES`` and ``KEEP_NODES`` take them, checked: caches of
    one layer [pages, ...] or of all [layers, pages, ...]."""
    if not isinstance(k_pages, torch.Tensor) or k_pages.ndim not in (4, 5):
        raise ValueError(f"{what}: k_pages must be [pages, kv_heads, page_size, head_dim], or that "
                         "per layer")
    if k_pages.ndim == 4:
        _check_cache(what, k_pages, v_pages, block_table)
        layers, k_layer, v_layer, k, v = 1, 0, 0, k_pages, v_pages
    else:
        if not isinstance(v_pages, torch.Tensor) or v_pages.shape != k_pages.shape or not len(k_pages):
            raise ValueError(f"{what}: v_pages must have k_pages' shape, of one layer at least")
        layers, k_layer, v_layer = k_pages.shape[0], k_pages.stride(0), v_pages.stride(0)
        k, v = k_pages[0], v_pages[0]
        _check_cache(what, k, v, block_table)
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            if layers > 1 and t.stride(0) < (t.shape[1] - 1) * t.stride(1) + k[0:1].numel():
                raise ValueError(f"{what}: {name}'s layers overlap")
    return (*k.shape, _outer_stride(k), _outer_stride(v), layers, k_layer, v_layer)


def _layers_of(what: str, k_pages, v_pages, block_table, *int32) -> tuple:
    """``(n_pages, kv, page, hd, k page stride, v page stride, layers, k and v layer stride)``, GPU,
    type code, and whether the tensors ``int32`` of the call were found packed and on that GPU."""
    try:
        dt, dev, ndim = k_pages.dtype, k_pages.get_device(), k_pages.ndim
        if (ndim in (4, 5) and dt in _HALVES and v_pages.shape == k_pages.shape
                and _plain(dev, dt, k_pages, v_pages) and block_table.ndim == 2
                and _plain(dev, torch.int32, block_table, *int32)):
            layers = k_pages.shape[0] if ndim == 5 else 1
            n_pages, kv, page, hd = k_pages.shape[-4:]
            one = kv * page * hd
            if layers and (hd == 64 or hd == 128):
                return (n_pages, kv, page, hd, one, one, layers, n_pages * one, n_pages * one), dev, dt, True
    except AttributeError:
        pass
    return (_check_layers(what, k_pages, v_pages, block_table), k_pages.get_device(), k_pages.dtype,
            False)


@functools.lru_cache(maxsize=None)
def _tree_ws_bytes(device: int, hd: int) -> int:
    return _native.lib().moe_tree_attention_workspace_size(hd)


@_on_first_device
def tree_attention_workspace(k_pages: torch.Tensor) -> torch.Tensor:
    """A workspace for :func:`tree_attention` calls on caches with this head_dim."""
    nbytes = _tree_ws_bytes(k_pages.get_device(), k_pages.shape[-1])
    return torch.zeros(nbytes, dtype=torch.uint8, device=k_pages.device)


@_on_first_device
def tree_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                   block_table: torch.Tensor, lengths: torch.Tensor, visible: torch.Tensor,
                   counts: torch.Tensor | None = None, scale: float | None = None,
                   out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of a tree of drafted tokens per sequence over its cached keys and values.

    ``q`` [sequences, nodes, heads, head_dim] (sequences and nodes may be strided); ``lengths`` int32
    [sequences]: cached positions before the tree, which every node sees; node i's own keys and
    values are at position ``lengths[b] + i`` (:func:`rope_append` with ``slots``).  ``visible`` int64
    [sequences, nodes, ceil(nodes / 64)] (may be expanded): bit ``i % 64`` of word ``i // 64`` is
    set where the node sees node i, itself included (:func:`tree_masks` makes it from parents).
    ``counts`` int32 [sequences]: the nodes that are there (None: all).  A row that sees nothing
    is zeros, and so are rows past ``counts`` and of sequences with a negative length.  The cache as in
    :func:`paged_attention`; at most 2048 sequences, 1024 nodes and a table of 2^30 positions.  ``scale`` defaults to ``head_dim ** -0.5``.  Returns
    [sequences, nodes, heads, head_dim]; ``out``, if given, must not share memory with ``q``.

    ``workspace``: a buffer from :func:`tree_attention_workspace`, as for :func:`paged_attention`.
    """
    what = "tree_attention"
    try:
        n_pages, kv, page, hd = k_pages.shape
        seqs, max_pages = block_table.shape
        _, nodes, heads, _ = q.shape
        words = (nodes + 63) // 64
        dt, dev = k_pages.dtype, k_pages.get_device()
        plain = (dt in _HALVES and (hd == 64 or hd == 128) and q.shape == (seqs, nodes, heads, hd)
                 and v_pages.shape == k_pages.shape and lengths.shape == (seqs,)
                 and visible.shape == (seqs, nodes, words)
                 and _plain(dev, dt, q, k_pages, v_pages)
                 and _plain(dev, torch.int32, lengths, block_table)
                 and _plain(dev, torch.int64, visible))
    except (AttributeError, ValueError):
        plain = False
    if not plain:
        _check_cache(what, k_pages, v_pages, block_table)
        n_pages, kv, page, hd = k_pages.shape
        dt, dev = k_pages.dtype, k_pages.get_device()
        seqs, max_pages = block_table.shape
        _serve_check(what, dev, ("q", q, dt, (seqs, None, None, hd), 2),
                     ("lengths", lengths, torch.int32, (seqs,), 1))
        nodes, heads = q.shape[1:3]
        words = (nodes + 63) // 64
        _serve_check(what, dev, ("visible", visible, torch.int64, (seqs, nodes, words), 1))
        if min(q.stride()) < 0 or min(visible.stride()) < 0:
            raise ValueError(f"{what}: strides must not be negative")
    if page % 16:
        raise ValueError(f"{what}: page_size must be a multiple of 16, got {page}")
    if heads == 0 or kv == 0 or heads % kv:
        raise ValueError(f"{what}: {heads} query heads do not divide over {kv} KV heads")
    if counts is not None:
        _serve_check(what, dev, ("counts", counts, torch.int32, (seqs,), 1))
    if out is None:
        out = torch.empty_like(q) if plain else q.new_empty((seqs, nodes, heads, hd))
    else:
        _serve_check(what, dev, ("out", out, dt, (seqs, nodes, heads, hd), 4))
    if seqs == 0 or nodes == 0:
        return out
    stream = _raw_stream(dev)
    nbytes = _tree_ws_bytes(dev, hd)
    if workspace is None:
        workspace = _serve_scratch(dev, stream, nbytes)
    else:
        _check_workspace(what, workspace, dev, nbytes)
    page_elems, row = kv * page * hd, heads * hd
    if plain:
        strides = (page_elems, page_elems, max_pages, nodes * row, row, nodes * words, words)
    else:
        node = q.stride(1) if nodes > 1 else row
        strides = (_outer_stride(k_pages), _outer_stride(v_pages), _outer_stride(block_table),
                   q.stride(0) if seqs > 1 else nodes * node, node, visible.stride(0),
                   visible.stride(1))
    status = _native.lib().moe_tree_attention(_native.TREE_ATTENTION.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), strides[0], strides[1], n_pages, kv, page, hd,
        _DTYPE_CODES[dt], block_table.data_ptr(), strides[2], seqs, max_pages, q.data_ptr(),
        strides[3], strides[4], nodes, heads, lengths.data_ptr(),
        0 if counts is None else counts.data_ptr(), visible.data_ptr(), strides[5], strides[6],
        hd ** -0.5 if scale is None else scale, out.data_ptr(), workspace.data_ptr(), nbytes, stream))
    if status:
        check(status, "moe_tree_attention")
    return out


def tree_masks(parents) -> torch.Tensor:
    """``visible`` of :func:`tree_attention` from a tree's parents: int64 [nodes, ceil(nodes / 64)] on
    the CPU.  ``parents[i] < i`` is node i's parent, -1 where it follows the cached tokens."""
    seen: list[int] = []
    for i, p in enumerate(parents):
        p = int(p)
        if not -1 <= p < i:
            raise ValueError(f"tree_masks: node {i}'s parent must be -1 to {i - 1}, got {p}")
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    words = (len(seen) + 63) // 64
    rows = [[(m >> 64 * w & (1 << 64) - 1) - (m >> 64 * w + 63 & 1) * (1 << 64) for w in range(words)]
            for m in seen]
    return torch.tensor(rows, dtype=torch.int64).view(len(seen), words)


@_on_first_device
def fork_pages(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
               lengths: torch.Tensor, parents: torch.Tensor, refs: torch.Tensor, room: int = 1,
               workspace: torch.Tensor | None = None) -> None:
    """Fork, end and grow the sequences of a paged cache, in place.

    Row i of ``block_table`` int32 [sequences, max_pages] becomes a copy of row ``parents[i]``
    (int32; i itself: it stays, -1: it ends and its pages are freed), ``lengths[i]`` int32 its
    parent's.  Then the pages of its next ``room`` positions become its own: a missing one is taken
    from the free pages, the lowest number first, and one that others list too is replaced by such a
    page with the filled positions copied, in every layer.  ``k_pages`` / ``v_pages``: as in
    :func:`rope_append`, or of all layers, [layers, pages, ...].  ``refs`` int32 [pages]: how many
    entries of the table name each page (0: free), kept up to date; a holder elsewhere (a prefix kept
    for later) adds one to keep its page from being written or freed.  Entries without a page are
    negative.  A row of a negative length is no sequence: it and its copies stay so and are given no
    page.  A row that ended has length 0: if later calls are to pass it over (a decode step would
    look for its first page) set its length below 0.  When no page is free the entry is -1, which
    shows in :func:`check_device`, as do parents and pages out of range and lengths past the table.

    ``workspace``: :func:`fork_pages_workspace`, as for :func:`paged_attention`.
    """
    what = "fork_pages"
    cache, dev, dt, plain = _layers_of(what, k_pages, v_pages, block_table, lengths, parents, refs)
    seqs, max_pages = block_table.shape
    if not (plain and lengths.shape == parents.shape == (seqs,) and refs.shape == cache[:1]):
        _serve_check(what, dev, ("lengths", lengths, torch.int32, (seqs,), 1),
                     ("parents", parents, torch.int32, (seqs,), 1),
                     ("refs", refs, torch.int32, cache[:1], 1))
        if seqs > 1 and block_table.stride(0) < max_pages:
            raise ValueError(f"{what}: block_table's rows overlap")
    stream = _raw_stream(dev)
    nbytes = _fork_ws_bytes(seqs)
    if workspace is None:
        workspace = _serve_scratch(dev, stream, nbytes)
    else:
        _check_workspace(what, workspace, dev, nbytes)
    n_pages, kv, page, hd, k_page, v_page, layers, k_layer, v_layer = cache
    status = _native.lib().moe_fork_pages(_native.FORK_PAGES.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), k_page, v_page, n_pages, kv, page, hd, _DTYPE_CODES[dt],
        block_table.data_ptr(), max_pages if plain else max(_outer_stride(block_table), max_pages),
        seqs, max_pages, layers, k_layer, v_layer, lengths.data_ptr(), parents.data_ptr(),
        refs.data_ptr(), room, workspace.data_ptr(), nbytes, stream))
    if status:
        check(status, "moe_fork_pages")


@functools.lru_cache(maxsize=1024)
def _fork_ws_bytes(seqs: int) -> int:
    return _native.lib().moe_fork_pages_workspace_size(seqs)


@_on_first_device
def fork_pages_workspace(block_table: torch.Tensor) -> torch.Tensor:
    """A workspace for :func:`fork_pages` calls on tables of as many rows."""
    nbytes = _fork_ws_bytes(block_table.shape[0])
    return torch.zeros(nbytes, dtype=torch.uint8, device=block_table.device)


@_on_first_device
def keep_nodes(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
               lengths: torch.Tensor, keep: torch.Tensor) -> torch.Tensor:
    """Move the accepted nodes of drafted trees to the end of their sequences; the new lengths.

    ``keep`` int32 [sequences, any number]: the accepted nodes' indices, rising, up to the first
    negative entry (rows may be strided).  In every layer the keys and values of position
    ``lengths[b] + keep[b, j]`` move to ``lengths[b] + j``; the cache as in :func:`fork_pages`.
    Returns ``lengths`` plus the kept nodes' number, int32 [sequences]; ``lengths[b] < 0`` is no
    sequence and stays.  A list that falls or has no pages ends there and shows in
    :func:`check_device`.  The pages moved in must be the sequence's own (:func:`fork_pages`).
    """
    what = "keep_nodes"
    cache, dev, dt, plain = _layers_of(what, k_pages, v_pages, block_table, lengths, keep)
    seqs, max_pages = block_table.shape
    if not (plain and lengths.shape == (seqs,) and keep.ndim == 2 and keep.shape[0] == seqs):
        _serve_check(what, dev, ("lengths", lengths, torch.int32, (seqs,), 1),
                     ("keep", keep, torch.int32, (seqs, None), 1))
    most = keep.shape[1]
    out = torch.empty_like(lengths)
    n_pages, kv, page, hd, k_page, v_page, layers, k_layer, v_layer = cache
    strides = ((max_pages, most) if plain or not seqs else (_outer_stride(block_table),
                                                            _outer_stride(keep)))
    status = _native.lib().moe_keep_nodes(_native.KEEP_NODES.pack(
        k_pages.data_ptr(), v_pages.data_ptr(), k_page, v_page, n_pages, kv, page, hd, _DTYPE_CODES[dt],
        block_table.data_ptr(), strides[0], seqs, max_pages, layers, k_layer, v_layer,
        lengths.data_ptr(), keep.data_ptr(), strides[1], most, out.data_ptr(), _raw_stream(dev)))
    if status:
        check(status, "moe_keep_nodes")
    return out


@functools.lru_cache(maxsize=1024)
def _beam_ws_bytes(device: int, groups: int, beams: int, vocab: int, count: int, code: int) -> int:
    return _native.lib().moe_beam_select_workspace_size(groups, beams, vocab, count, code)


@_on_first_device
def beam_select(logits: torch.Tensor, scores: torch.Tensor, count: int | None = None,
                workspace: torch.Tensor | None = None):
    """``(scores fp32, parents int32, tokens int64)``, each [groups, count]: every group's best
    continuations over its beams and the vocabulary, the best first.

    ``logits`` [groups * beams, vocab], fp16, bf16 or fp32 (rows may be strided, or one row expanded;
    vocab <= 2^20); ``scores`` fp32 [groups, beams]: the beams' running sums of log-probabilities, -inf
    for a beam that is not there (as all but one are at the first step); ``count`` (default: beams)
    and beams at most 64.  A continuation scores its beam's score plus the token's log-probability;
    ``parents`` is the beam's index in its group.  Equal scores go to the lower beam, in a beam to the
    larger logit, then the lower token.  Tokens at -inf are no candidates, NaN logits count as
    -inf; places without a candidate hold (-inf, 0, 0).  A beam that has ended is carried along by a
    row that is -inf but for its end token.

    ``workspace``: a zeroed buffer of :func:`beam_select_workspace` that no call on another stream
    uses at the same time, as for :func:`paged_attention`; one made for the largest batch and count
    serves the smaller ones.
    """
    what = "beam_select"
    if not isinstance(logits, torch.Tensor) or logits.ndim != 2:
        raise ValueError(f"{what}: logits must be [groups * beams, vocab]")
    code = _DTYPE_CODES.get(logits.dtype)
    if code is None:
        raise ValueError(f"{what}: logits must be float16, bfloat16 or float32, got {logits.dtype}")
    if not isinstance(scores, torch.Tensor) or scores.ndim != 2:
        raise ValueError(f"{what}: scores must be [groups, beams]")
    dev = logits.get_device()
    rows, vocab = logits.shape
    groups, beams = scores.shape
    if not (_plain(dev, torch.float32, scores) and logits.stride(1) == 1):
        _serve_check(what, dev, ("logits", logits, logits.dtype, logits.shape, 1),
                     ("scores", scores, torch.float32, scores.shape, 2))
    if rows != groups * beams:
        raise ValueError(f"{what}: logits has {rows} rows for {groups} groups of {beams} beams")
    if count is None:
        count = beams
    if not (1 <= beams <= 64 and 1 <= count <= 64):
        raise ValueError(f"{what}: 1 to 64 beams and 1 to 64 continuations are served, got {beams} "
                         f"and {count}")
    like = scores if count == beams else scores.new_empty((groups, count))
    out = (torch.empty_like(like) if like is scores else like, torch.empty_like(like, dtype=torch.int32),
           torch.empty_like(like, dtype=torch.int64))
    stream = _raw_stream(dev)
    nbytes = _beam_ws_bytes(dev, groups, beams, vocab, count, code)
    if workspace is None:
        workspace = _serve_scratch(dev, stream, nbytes)
    else:
        _check_workspace(what, workspace, dev, nbytes)
    status = _native.lib().moe_beam_select(_native.BEAM_SELECT.pack(
        logits.data_ptr(), _outer_stride(logits), groups, beams, vocab, code, scores.data_ptr(), count,
        out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), workspace.data_ptr(), nbytes, stream))
    if status:
        check(status, "moe_beam_select")
    return out


@_on_first_device
def beam_select_workspace(logits: torch.Tensor, beams: int, count: int | None = None) -> torch.Tensor:
    """A workspace for :func:`beam_select` calls on up to as many rows of logits, and up to ``count``."""
    rows, vocab = logits.shape
    nbytes = _beam_ws_bytes(logits.get_device(), rows // beams, beams, vocab,
                            beams if count is None else count, _DTYPE_CODES[logits.dtype])
    return torch.zeros(nbytes, dtype=torch.uint8, device=logits.device)
