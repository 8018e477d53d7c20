"""The operator surface of the reference's pybind11 module `sparsebench._C`
(csrc/bindings.cpp:5-16, csrc/ops.hpp:11-36), over the gfx950 C ABI.

Same four functions, same keyword names, same outputs, and the same
RuntimeError messages for bad arguments (the checks of csrc/routing.cu:198-224,
csrc/sdd.cu:126-153, csrc/dsd.cpp:29-61, csrc/dsd_v5.cu:108-110,
csrc/smoke.cu:24), in the same order. Outputs come from torch's caching
allocator on the input's device and all work is enqueued on torch's current
stream, so nothing here syncs and every call can be captured in a graph.

combine_cuda is this build's addition: the combine step of moe_forward as one
kernel.
"""

from __future__ import annotations

import array
import contextlib
import ctypes
import functools
import itertools
import operator

import torch

from sparsebench_amd._lib import check, lib, stream_of

_I32_MAX = 2**31 - 1
_MAX_EXPERTS = 1024
_DSD_TILE_N = 128
# dsd version code -> dead row blocks written as zeros (versions 1-3) or left unwritten (4 on)
_DSD_VERSIONS = {1: True, 2: True, 21: True, 3: True, 31: True, 4: False, 41: False, 5: False}
_GATE_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _fail(msg: str) -> None:
    raise RuntimeError(msg)


def _shape(t: torch.Tensor) -> str:
    return "[" + ", ".join(str(s) for s in t.shape) + "]"


def _check_index(t: torch.Tensor, name: str) -> None:
    if not (t.is_cuda and t.dtype == torch.int32 and t.dim() == 1 and t.is_contiguous()):
        _fail(f"{name} must be a contiguous 1-D int32 CUDA tensor")


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


_TEST_HOOKS = {"expert_gate": 0, "topk_kernel": 1}


def set_test_hook(name: str, value: int) -> None:
    """Forces one of the library's own choices for tests (include/sparsebench_hip.h:
    expert_gate 1 = expert tiles, 2 = row blocks; topk_kernel 1 = wave form,
    2 = lane form); 0 restores the choice."""
    if name not in _TEST_HOOKS:
        raise ValueError(f"unknown test hook {name!r}")
    check(lib().sb_set_test_hook(_TEST_HOOKS[name], int(value)))


def arch_probe(n: int) -> torch.Tensor:
    """int32[n] filled with the architecture number of the code that ran (950 on gfx950)."""
    if n <= 0:
        _fail(f"arch_probe: n must be positive, got {n}")
    out = torch.empty(n, dtype=torch.int32, device="cuda")
    check(lib().sb_arch_probe(out.data_ptr(), n, stream_of(out.device)))
    return out


def routing_sizes(num_copies: int, num_experts: int, ffn_dim: int, block_size: int) -> tuple[int, int, int]:
    """(max_row_blocks, max_rows, workspace int32 elements) for n = T*k copies."""
    rb, rows, ws = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
    check(lib().sb_routing_sizes(num_copies, num_experts, ffn_dim, block_size,
                                 ctypes.byref(rb), ctypes.byref(rows), ctypes.byref(ws)))
    return rb.value, rows.value, ws.value


def build_topology_cuda(
    expert_idx: torch.Tensor,
    num_experts: int,
    ffn_dim: int,
    block_size: int,
    valid_tokens: torch.Tensor | None = None,
) -> list[torch.Tensor]:
    """Routing -> block-sparse layout on the GPU, no host sync.

    Returns, in order: tokens_per_expert [E], padded_offsets [E+1],
    row_token [max_rows], copy_row [T*k], row_block_expert [max_row_blocks],
    row_offsets [max_row_blocks+1], col_indices [max_row_blocks*ffn_blocks],
    error [1] (all int32; csrc/ops.hpp:13-21).

    valid_tokens (this build's extension, default None = reference behaviour):
    an int32 CUDA scalar T' <= T; copies of tokens >= T' are ignored.
    """
    if not expert_idx.is_cuda:
        _fail("expert_idx must be a CUDA tensor")
    if expert_idx.dim() != 2 or expert_idx.shape[0] == 0 or expert_idx.shape[1] == 0:
        _fail(f"expert_idx must be [T, k] with T, k > 0, got {_shape(expert_idx)}")
    if expert_idx.dtype not in (torch.int32, torch.int64):
        _fail(f"expert_idx must be int32 or int64, got {expert_idx.dtype}")
    if not expert_idx.is_contiguous():
        _fail("expert_idx must be contiguous")
    if not 0 < num_experts <= _MAX_EXPERTS:
        _fail(f"num_experts must be in [1, {_MAX_EXPERTS}], got {num_experts}")
    if not 0 < block_size <= _I32_MAX:
        _fail("block_size must be in [1, 2^31)")
    if ffn_dim <= 0 or ffn_dim % block_size != 0:
        _fail(f"ffn_dim ({ffn_dim}) must be a positive multiple of block_size ({block_size})")
    num_tokens, k = expert_idx.shape
    n = num_tokens * k
    # Worst case: every expert wastes block_size - 1 rows (csrc/routing.cu:213-224).
    max_row_blocks = (n + num_experts * (block_size - 1)) // block_size
    max_rows = max_row_blocks * block_size
    ffn_blocks = ffn_dim // block_size
    if max_rows > _I32_MAX // ffn_dim or max_row_blocks * ffn_blocks >= _I32_MAX or n > _I32_MAX:
        _fail("problem too large for int32 indexing")
    if valid_tokens is not None:
        if not (valid_tokens.is_cuda and valid_tokens.dtype == torch.int32 and valid_tokens.numel() == 1):
            _fail("valid_tokens must be a one-element int32 CUDA tensor")

    dev = expert_idx.device
    opts = {"dtype": torch.int32, "device": dev}
    num_chunks = (n + 1023) // 1024
    workspace = torch.empty(num_chunks * (num_experts + 1), **opts)
    tokens_per_expert = torch.empty(num_experts, **opts)
    padded_offsets = torch.empty(num_experts + 1, **opts)
    row_token = torch.empty(max_rows, **opts)
    copy_row = torch.empty(n, **opts)
    row_block_expert = torch.empty(max_row_blocks, **opts)
    row_offsets = torch.empty(max_row_blocks + 1, **opts)
    col_indices = torch.empty(max_row_blocks * ffn_blocks, **opts)
    error = torch.empty(1, **opts)
    check(lib().sb_routing(
        expert_idx.data_ptr(), 1 if expert_idx.dtype == torch.int64 else 0, num_tokens, k, num_experts, ffn_dim,
        block_size, _ptr(valid_tokens), workspace.data_ptr(), tokens_per_expert.data_ptr(),
        padded_offsets.data_ptr(), row_token.data_ptr(), copy_row.data_ptr(), row_block_expert.data_ptr(),
        row_offsets.data_ptr(), col_indices.data_ptr(), error.data_ptr(), stream_of(dev),
    ))
    return [tokens_per_expert, padded_offsets, row_token, copy_row, row_block_expert, row_offsets, col_indices, error]


def sdd_cuda(
    x: torch.Tensor,
    w1: torch.Tensor,
    row_token: torch.Tensor,
    row_block_expert: torch.Tensor,
    row_offsets: torch.Tensor,
    num_nnz: int,
    apply_gelu: bool,
) -> torch.Tensor:
    """H blocks [num_nnz, 128, 128] bf16 = (gelu)(x[row_token] @ w1[expert]) on the layout's blocks."""
    if not (x.is_cuda and w1.is_cuda and x.device == w1.device):
        _fail("x and w1 must be on the same GPU")
    if x.dtype != torch.bfloat16 or w1.dtype != torch.bfloat16:
        _fail("x and w1 must be bfloat16")
    if not (x.is_contiguous() and w1.is_contiguous()):
        _fail("x and w1 must be contiguous")
    if not (x.dim() == 2 and w1.dim() == 3 and w1.shape[1] == x.shape[1]):
        _fail(f"x must be [T, D] and w1 [E, D, F], got {_shape(x)} and {_shape(w1)}")
    _check_index(row_token, "row_token")
    _check_index(row_block_expert, "row_block_expert")
    _check_index(row_offsets, "row_offsets")
    if x.data_ptr() % 16 or w1.data_ptr() % 16:
        _fail("x and w1 must be 16-byte aligned")
    d_model, ffn_dim = x.shape[1], w1.shape[2]
    num_row_blocks = row_offsets.numel() - 1
    if d_model <= 0 or d_model % 64:
        _fail(f"sdd needs D ({d_model}) to be a multiple of 64")
    if ffn_dim <= 0 or ffn_dim % 256:
        _fail(f"sdd needs F ({ffn_dim}) to be a multiple of 256")
    if row_token.numel() != num_row_blocks * 128:
        _fail(f"sdd needs block size 128: row_token has {row_token.numel()} rows for {num_row_blocks} row blocks")
    if row_block_expert.numel() != num_row_blocks:
        _fail("row_block_expert must have one entry per row block")
    if num_nnz != num_row_blocks * (ffn_dim // 128):
        _fail(f"expected {num_row_blocks * (ffn_dim // 128)} blocks (row blocks x F/128), got {num_nnz}")
    if num_row_blocks * (ffn_dim // 256) > _I32_MAX or ffn_dim * d_model > _I32_MAX:
        _fail("problem too large")
    out = torch.empty(num_nnz, 128, 128, dtype=w1.dtype, device=w1.device)
    if num_row_blocks <= 0:
        return out
    check(lib().sb_sdd(
        x.data_ptr(), w1.data_ptr(), row_token.data_ptr(), row_block_expert.data_ptr(), row_offsets.data_ptr(),
        out.data_ptr(), x.shape[0], d_model, ffn_dim, w1.shape[0], num_row_blocks, 1 if apply_gelu else 0,
        stream_of(x.device),
    ))
    return out


def dsd_cuda(
    blocks: torch.Tensor, w: torch.Tensor, row_offsets: torch.Tensor, col_indices: torch.Tensor, version: int,
    routed: bool = False,
) -> torch.Tensor:
    """out [(len(row_offsets)-1)*bs, D] bf16 = BSR(blocks, row_offsets, col_indices) @ w.

    Every version code of the reference is accepted and gives the same
    results; codes 1, 2, 21, 3, 31 write dead row blocks as zeros, codes 4,
    41, 5 leave them unwritten, and 5 needs block size 128 and D % 256 == 0.

    routed (this build's extension): the arrays are a routing layout, so the
    kernel may take its row blocks in pairs; the results are the same.
    """
    if not (blocks.is_cuda and w.is_cuda):
        _fail("blocks and w must be CUDA tensors")
    if not (blocks.device == w.device and row_offsets.device == w.device and col_indices.device == w.device):
        _fail("all inputs must be on the same GPU")
    if blocks.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
        _fail("blocks and w must be bfloat16")
    if not (blocks.is_contiguous() and w.is_contiguous()):
        _fail("blocks and w must be contiguous")
    if not (blocks.dim() == 3 and blocks.shape[1] == blocks.shape[2]):
        _fail(f"blocks must be [nnz, bs, bs], got {_shape(blocks)}")
    if w.dim() != 2:
        _fail(f"w must be [E*F, D], got {_shape(w)}")
    _check_index(row_offsets, "row_offsets")
    _check_index(col_indices, "col_indices")
    bs, d_model = blocks.shape[1], w.shape[1]
    num_row_blocks = row_offsets.numel() - 1
    if bs not in (64, 128):
        _fail(f"block size must be 64 or 128, got {bs}")
    if d_model <= 0 or d_model % _DSD_TILE_N:
        _fail(f"D ({d_model}) must be a positive multiple of {_DSD_TILE_N}")
    if d_model // _DSD_TILE_N > 65535:
        _fail("D too large for grid y")
    if w.shape[0] % bs:
        _fail(f"w rows ({w.shape[0]}) must be a multiple of the block size ({bs})")
    if num_row_blocks < 0:
        _fail("row_offsets must have at least one entry")
    if blocks.shape[0] != col_indices.numel():
        _fail(f"blocks has {blocks.shape[0]} blocks but col_indices has {col_indices.numel()}")
    if num_row_blocks * bs > _I32_MAX:
        _fail("too many row blocks")
    if num_row_blocks * (d_model // _DSD_TILE_N) > _I32_MAX:
        _fail("too many tiles for a 1-D grid")
    if blocks.data_ptr() % 16:
        _fail("blocks must be 16-byte aligned")
    if w.data_ptr() % 16:
        _fail("w must be 16-byte aligned")
    out = torch.empty(num_row_blocks * bs, d_model, dtype=w.dtype, device=w.device)
    if num_row_blocks == 0:
        return out
    if version not in _DSD_VERSIONS:
        _fail(f"unknown dsd version {version}")
    if version == 5 and (bs != 128 or d_model % 256):
        _fail(f"dsd v5 needs block size 128 and D a multiple of 256, got block size {bs}, D {d_model}")
    launch = lib().sb_dsd_routed if routed else lib().sb_dsd
    check(launch(
        blocks.data_ptr(), w.data_ptr(), row_offsets.data_ptr(), col_indices.data_ptr(), out.data_ptr(),
        blocks.shape[0], w.shape[0], num_row_blocks, bs, d_model, 1 if _DSD_VERSIONS[version] else 0,
        stream_of(w.device),
    ))
    return out


def _check_expert_layout(topo, device: torch.device) -> None:
    if topo.block_size != 128:
        _fail(f"expert tiles need block size 128, got {topo.block_size}")
    for name in ("tokens_per_expert", "padded_offsets", "row_token", "row_block_expert", "row_offsets", "col_indices"):
        t = getattr(topo, name)
        _check_index(t, name)
        if t.device != device:
            _fail("all inputs must be on the same GPU")
    if topo.padded_offsets.numel() != topo.num_experts + 1 or topo.tokens_per_expert.numel() != topo.num_experts:
        _fail("tokens_per_expert / padded_offsets do not match the expert count")
    max_row_blocks = topo.row_token.numel() // 128
    if (topo.row_token.numel() != max_row_blocks * 128 or topo.row_block_expert.numel() != max_row_blocks
            or topo.row_offsets.numel() != max_row_blocks + 1
            or topo.col_indices.numel() != max_row_blocks * topo.ffn_blocks):
        _fail("the routing layout's arrays do not have worst-case sizes of one layout")


def sdd_experts_cuda(x: torch.Tensor, w1: torch.Tensor, topo, apply_gelu: bool) -> torch.Tensor:
    """SDD of the MoE layer (this build's addition): expert-major tiles when
    the routing is balanced, else row-block tiles, chosen on the GPU; for
    F % 512 != 0, each expert's row blocks in pairs (every row written).

    topo: a routing layout from route_device / route_assigned / route_rounded.
    Returns H blocks [max_row_blocks*F/128, 128, 128] bf16 whose real rows are
    bit-identical to sdd_cuda's; padding rows past each expert's last 32-row
    group may be left unwritten (the layer never reads them).
    """
    if not (x.is_cuda and w1.is_cuda and x.device == w1.device):
        _fail("x and w1 must be on the same GPU")
    if x.dtype != torch.bfloat16 or w1.dtype != torch.bfloat16:
        _fail("x and w1 must be bfloat16")
    if not (x.is_contiguous() and w1.is_contiguous()):
        _fail("x and w1 must be contiguous")
    if not (x.dim() == 2 and w1.dim() == 3 and w1.shape[1] == x.shape[1]):
        _fail(f"x must be [T, D] and w1 [E, D, F], got {_shape(x)} and {_shape(w1)}")
    _check_expert_layout(topo, x.device)
    num_experts, d_model, ffn_dim = w1.shape
    if num_experts != topo.num_experts or ffn_dim != topo.ffn_blocks * 128:
        _fail("w1 does not match the routing layout")
    max_row_blocks = topo.row_token.numel() // 128
    out = torch.empty(max_row_blocks * (ffn_dim // 128), 128, 128, dtype=w1.dtype, device=w1.device)
    check(lib().sb_sdd_experts(
        x.data_ptr(), w1.data_ptr(), topo.row_token.data_ptr(), topo.row_block_expert.data_ptr(),
        topo.row_offsets.data_ptr(), topo.tokens_per_expert.data_ptr(), topo.padded_offsets.data_ptr(),
        out.data_ptr(), x.shape[0], d_model, ffn_dim, num_experts, max_row_blocks, 1 if apply_gelu else 0,
        stream_of(x.device),
    ))
    return out


def dsd_experts_cuda(h: torch.Tensor, w2_cat: torch.Tensor, topo) -> torch.Tensor:
    """DSD (version 5) of the MoE layer (this build's addition): expert-major
    tiles when the routing is balanced, else the per-row-block kernel, chosen
    on the GPU.

    h: sdd_experts_cuda's (or sdd_cuda's) blocks on topo's layout; w2_cat
    [E*F, D]. Returns y [max_row_blocks*128, D] bf16 whose real rows are
    bit-identical to dsd_cuda's; padding rows may be left unwritten.
    """
    if not (h.is_cuda and w2_cat.is_cuda and h.device == w2_cat.device):
        _fail("h and w must be on the same GPU")
    if h.dtype != torch.bfloat16 or w2_cat.dtype != torch.bfloat16:
        _fail("h and w must be bfloat16")
    if not (h.is_contiguous() and w2_cat.is_contiguous()):
        _fail("h and w must be contiguous")
    _check_expert_layout(topo, h.device)
    max_row_blocks = topo.row_token.numel() // 128
    ffn_dim = topo.ffn_blocks * 128
    if h.dim() != 3 or h.shape != (max_row_blocks * topo.ffn_blocks, 128, 128):
        _fail(f"h must be [{max_row_blocks * topo.ffn_blocks}, 128, 128] for this layout, got {_shape(h)}")
    if w2_cat.dim() != 2 or w2_cat.shape[0] != topo.num_experts * ffn_dim:
        _fail(f"w must be [E*F, D] = [{topo.num_experts * ffn_dim}, D], got {_shape(w2_cat)}")
    d_model = w2_cat.shape[1]
    out = torch.empty(max_row_blocks * 128, d_model, dtype=w2_cat.dtype, device=w2_cat.device)
    check(lib().sb_dsd_experts(
        h.data_ptr(), w2_cat.data_ptr(), topo.tokens_per_expert.data_ptr(), topo.padded_offsets.data_ptr(),
        topo.row_block_expert.data_ptr(), topo.row_offsets.data_ptr(), topo.col_indices.data_ptr(), out.data_ptr(),
        max_row_blocks, topo.num_experts, topo.copy_row.numel(), ffn_dim, d_model, stream_of(h.device),
    ))
    return out


def expert_tiles_fit(d_model: int, ffn_dim: int, max_row_blocks: int) -> bool:
    """Whether sdd_experts_cuda / dsd_experts_cuda take this shape (else the per-row-block kernels)."""
    h_bytes = max_row_blocks * (ffn_dim // 128) * 128 * 128 * 2
    return (d_model % 256 == 0 and ffn_dim % 256 == 0 and h_bytes < 2**31 and ffn_dim * d_model * 2 < 2**31)


def combine_cuda(
    y: torch.Tensor,
    copy_row: torch.Tensor,
    expert_weight: torch.Tensor,
    valid_tokens: torch.Tensor | None = None,
) -> torch.Tensor:
    """out [T, D] bf16: each token's k rows of y, gate-weighted, summed in fp32.

    y [rows, D] bf16, copy_row [T*k] int32 (row of copy t*k+j, -1 = skipped),
    expert_weight [T, k] bf16/fp16/fp32. Rows t >= valid_tokens (if given) are
    left unwritten.
    """
    if not (y.is_cuda and copy_row.is_cuda and expert_weight.is_cuda):
        _fail("y, copy_row and expert_weight must be CUDA tensors")
    if y.dtype != torch.bfloat16 or y.dim() != 2 or not y.is_contiguous():
        _fail(f"y must be a contiguous [rows, D] bfloat16 tensor, got {_shape(y)} {y.dtype}")
    _check_index(copy_row, "copy_row")
    if expert_weight.dim() != 2 or expert_weight.numel() != copy_row.numel():
        _fail(f"expert_weight must be [T, k] with T*k == len(copy_row), got {_shape(expert_weight)}")
    gates = expert_weight if expert_weight.dtype in _GATE_DTYPES else expert_weight.float()
    gates = gates.contiguous()
    num_tokens, k = expert_weight.shape
    out = torch.empty(num_tokens, y.shape[1], dtype=y.dtype, device=y.device)
    if num_tokens == 0:
        return out
    check(lib().sb_combine(
        y.data_ptr(), copy_row.data_ptr(), gates.data_ptr(), _GATE_DTYPES[gates.dtype], out.data_ptr(),
        num_tokens, k, y.shape[1], y.shape[0], _ptr(valid_tokens), stream_of(y.device),
    ))
    return out


# ---- routing given as assignments; router (this build's C ABI, no pybind11
# counterpart in the reference: there these steps are torch code in
# sparsebench/moe.py:59-91 and sparsebench/token_rounding.py) ----


def _check_copy_list(t: torch.Tensor, name: str) -> None:
    if not (t.is_cuda and t.dim() == 1 and t.dtype in (torch.int32, torch.int64) and t.is_contiguous()):
        _fail(f"{name} must be a contiguous 1-D int32 or int64 CUDA tensor")


def build_topology_assigned_cuda(
    token_of_copy: torch.Tensor,
    expert_of_copy: torch.Tensor,
    num_tokens: int,
    num_experts: int,
    ffn_dim: int,
    block_size: int,
    valid_tokens: torch.Tensor | None = None,
) -> list[torch.Tensor]:
    """The routing of a flat list (copy c: token_of_copy[c] -> expert_of_copy[c]),
    as build_topology_cuda with k = 1 and row_token holding token ids.
    Same 8 outputs, sized for N = len(list). No host sync."""
    _check_copy_list(token_of_copy, "token_of_copy")
    _check_copy_list(expert_of_copy, "expert_of_copy")
    n = expert_of_copy.numel()
    if token_of_copy.numel() != n or n == 0:
        _fail("token_of_copy and expert_of_copy must be non-empty and of the same length")
    if token_of_copy.device != expert_of_copy.device:
        _fail("token_of_copy and expert_of_copy must be on the same GPU")
    if not 0 < num_tokens <= _I32_MAX:
        _fail(f"num_tokens must be in [1, 2^31), got {num_tokens}")
    if valid_tokens is not None:
        if not (valid_tokens.is_cuda and valid_tokens.dtype == torch.int32 and valid_tokens.numel() == 1):
            _fail("valid_tokens must be a one-element int32 CUDA tensor")
    max_row_blocks, max_rows, ws = routing_sizes(n, num_experts, ffn_dim, block_size)
    dev = expert_of_copy.device
    opts = {"dtype": torch.int32, "device": dev}
    workspace = torch.empty(ws, **opts)
    outs = [torch.empty(num_experts, **opts), torch.empty(num_experts + 1, **opts), torch.empty(max_rows, **opts),
            torch.empty(n, **opts), torch.empty(max_row_blocks, **opts), torch.empty(max_row_blocks + 1, **opts),
            torch.empty(max_row_blocks * (ffn_dim // block_size), **opts), torch.empty(1, **opts)]
    check(lib().sb_routing_assigned(
        expert_of_copy.data_ptr(), 1 if expert_of_copy.dtype == torch.int64 else 0, token_of_copy.data_ptr(),
        1 if token_of_copy.dtype == torch.int64 else 0, n, num_tokens, num_experts, ffn_dim, block_size,
        _ptr(valid_tokens), workspace.data_ptr(), *(o.data_ptr() for o in outs), stream_of(dev),
    ))
    return outs


def token_csr_cuda(token_of_copy: torch.Tensor, copy_row: torch.Tensor, num_tokens: int
                   ) -> tuple[torch.Tensor, torch.Tensor]:
    """(token_offsets [T+1], token_copies [N]): each token's routed copies in
    ascending copy order. Deterministic, no host sync."""
    _check_copy_list(token_of_copy, "token_of_copy")
    _check_index(copy_row, "copy_row")
    n = token_of_copy.numel()
    if copy_row.numel() != n or n == 0:
        _fail("copy_row must have one entry per copy")
    dev = token_of_copy.device
    offsets = torch.empty(num_tokens + 1, dtype=torch.int32, device=dev)
    copies = torch.empty(n, dtype=torch.int32, device=dev)
    check(lib().sb_token_csr(token_of_copy.data_ptr(), 1 if token_of_copy.dtype == torch.int64 else 0,
                             copy_row.data_ptr(), n, num_tokens, offsets.data_ptr(), copies.data_ptr(),
                             stream_of(dev)))
    return offsets, copies


def combine_assigned_cuda(
    y: torch.Tensor,
    copy_row: torch.Tensor,
    weight_of_copy: torch.Tensor,
    token_offsets: torch.Tensor,
    token_copies: torch.Tensor | None,
    num_tokens: int,
    valid_tokens: torch.Tensor | None = None,
) -> torch.Tensor:
    """out [T, D] bf16: out[t] = sum over t's copies c (token_copies[token_offsets[t]:
    token_offsets[t+1]], or c = the index itself when token_copies is None) of
    fp32(y[copy_row[c]]) * fp32(weight_of_copy[c]), fp32 sum in copy order; 0 for
    a token with no copy."""
    if not (y.is_cuda and copy_row.is_cuda and weight_of_copy.is_cuda):
        _fail("y, copy_row and weight_of_copy must be CUDA tensors")
    if y.dtype != torch.bfloat16 or y.dim() != 2 or not y.is_contiguous():
        _fail(f"y must be a contiguous [rows, D] bfloat16 tensor, got {_shape(y)} {y.dtype}")
    _check_index(copy_row, "copy_row")
    _check_index(token_offsets, "token_offsets")
    if token_copies is not None:
        _check_index(token_copies, "token_copies")
    if token_offsets.numel() != num_tokens + 1:
        _fail(f"token_offsets must have T+1 = {num_tokens + 1} entries, got {token_offsets.numel()}")
    if weight_of_copy.dim() != 1 or weight_of_copy.numel() < copy_row.numel():
        _fail("weight_of_copy must be 1-D with one entry per copy")
    weights = weight_of_copy if weight_of_copy.dtype in _GATE_DTYPES else weight_of_copy.float()
    weights = weights.contiguous()
    out = torch.empty(num_tokens, y.shape[1], dtype=y.dtype, device=y.device)
    if num_tokens == 0:
        return out
    check(lib().sb_combine_assigned(
        y.data_ptr(), copy_row.data_ptr(), weights.data_ptr(), _GATE_DTYPES[weights.dtype], token_offsets.data_ptr(),
        _ptr(token_copies), out.data_ptr(), num_tokens, y.shape[1], y.shape[0], _ptr(valid_tokens),
        stream_of(y.device),
    ))
    return out


def _check_scores(scores: torch.Tensor) -> None:
    if not (scores.is_cuda and scores.dtype == torch.float32 and scores.dim() == 2 and scores.is_contiguous()):
        _fail("scores must be a contiguous [T, E] float32 CUDA tensor")
    if scores.shape[0] == 0 or scores.shape[1] == 0:
        _fail(f"scores must be [T, E] with T, E > 0, got {_shape(scores)}")


def router_topk_cuda(scores: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(top_idx [T, k] int32, top_weight [T, k] fp32): the k best experts of each
    token, best first (equal scores: lower expert first), and the picked
    scores over their sum."""
    _check_scores(scores)
    num_tokens, num_experts = scores.shape
    idx = torch.empty(num_tokens, k, dtype=torch.int32, device=scores.device)
    weight = torch.empty(num_tokens, k, dtype=torch.float32, device=scores.device)
    check(lib().sb_router_topk(scores.data_ptr(), num_tokens, num_experts, k, idx.data_ptr(), weight.data_ptr(),
                               stream_of(scores.device)))
    return idx, weight


def router_sizes(num_tokens: int, num_experts: int, k: int, tile: int, block_size: int, ffn_dim: int
                 ) -> tuple[int, int, int, int]:
    """(list capacity, max_row_blocks, max_rows, workspace int32 elements) of token rounding."""
    cap, rb, rows, ws = ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64(), ctypes.c_int64()
    check(lib().sb_router_sizes(num_tokens, num_experts, k, tile, block_size, ffn_dim, ctypes.byref(cap),
                                ctypes.byref(rb), ctypes.byref(rows), ctypes.byref(ws)))
    return cap.value, rb.value, rows.value, ws.value


def token_rounding_cuda(scores: torch.Tensor, k: int, tile: int, ffn_dim: int, block_size: int
                        ) -> dict[str, torch.Tensor]:
    """Token rounding fused with routing, no host sync. Returns the list
    (token_of_copy / expert_of_copy int32, weight_of_copy fp32, capacity-sized,
    -1 / -1 / 0 past the end), num_assignments [1], token_offsets [T+1], and the
    8 routing outputs of build_topology_assigned_cuda for that list."""
    _check_scores(scores)
    num_tokens, num_experts = scores.shape
    cap, max_row_blocks, max_rows, ws = router_sizes(num_tokens, num_experts, k, tile, block_size, ffn_dim)
    dev = scores.device
    i32 = {"dtype": torch.int32, "device": dev}
    out = {
        "token_of_copy": torch.empty(cap, **i32),
        "expert_of_copy": torch.empty(cap, **i32),
        "weight_of_copy": torch.empty(cap, dtype=torch.float32, device=dev),
        "num_assignments": torch.empty(1, **i32),
        "token_offsets": torch.empty(num_tokens + 1, **i32),
        "tokens_per_expert": torch.empty(num_experts, **i32),
        "padded_offsets": torch.empty(num_experts + 1, **i32),
        "row_token": torch.empty(max_rows, **i32),
        "copy_row": torch.empty(cap, **i32),
        "row_block_expert": torch.empty(max_row_blocks, **i32),
        "row_offsets": torch.empty(max_row_blocks + 1, **i32),
        "col_indices": torch.empty(max_row_blocks * (ffn_dim // block_size), **i32),
        "error": torch.empty(1, **i32),
    }
    workspace = torch.empty(ws, **i32)
    check(lib().sb_token_rounding(
        scores.data_ptr(), num_tokens, num_experts, k, tile, block_size, ffn_dim, workspace.data_ptr(),
        *(t.data_ptr() for t in out.values()), stream_of(dev),
    ))
    return out


# ---- the whole layer in one call (this build's C ABI): moe_forward and its
# variants without stage marks ----

_INDEX_DTYPES = {torch.int32: 0, torch.int64: 1}


@functools.lru_cache(maxsize=256)
def layer_bytes(num_tokens: int, num_copies: int, num_experts: int, d_model: int, ffn_dim: int) -> int | None:
    """Workspace bytes of layer_cuda (num_tokens = 0) or layer_assigned_cuda; None for a
    shape that the stages must take one by one (or refuse)."""
    size = ctypes.c_int64()
    if lib().sb_layer_sizes(num_tokens, num_copies, num_experts, d_model, ffn_dim, ctypes.byref(size)):
        return None
    return size.value


@functools.lru_cache(maxsize=256)
def layer_rounded_bytes(num_tokens: int, num_experts: int, k: int, tile: int, d_model: int, ffn_dim: int
                        ) -> int | None:
    """As layer_bytes, for layer_rounded_cuda."""
    size = ctypes.c_int64()
    if lib().sb_layer_rounded_sizes(num_tokens, num_experts, k, tile, d_model, ffn_dim, ctypes.byref(size)):
        return None
    return size.value


def _layer_operands_ok(x: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor) -> bool:
    """Whether the operands pass every check of the stages (which the caller falls back to, for their message)."""
    dev = x.device
    return (dev.type == "cuda" and w1.device == dev and w2.device == dev
            and x.dtype is torch.bfloat16 and w1.dtype is torch.bfloat16 and w2.dtype is torch.bfloat16
            and x.dim() == 2 and x.is_contiguous() and w1.is_contiguous() and w2.is_contiguous()
            and not (x.data_ptr() | w1.data_ptr() | w2.data_ptr()) % 16)


def _valid_tokens_ok(valid_tokens: torch.Tensor | None) -> bool:
    return valid_tokens is None or (
        valid_tokens.is_cuda and valid_tokens.dtype is torch.int32 and valid_tokens.numel() == 1)


def layer_cuda(x: torch.Tensor, expert_idx: torch.Tensor, expert_weight: torch.Tensor, w1: torch.Tensor,
               w2: torch.Tensor, valid_tokens: torch.Tensor | None) -> torch.Tensor | None:
    """moe_forward's four stages as one call, or None when some operand or the
    shape is not one that they all take as it is (then the stages say why).
    Shapes are moe_forward's, checked there."""
    num_experts, d_model, ffn_dim = w1.shape
    num_tokens, k = x.shape[0], expert_idx.shape[-1]
    idx_code, gate_code = _INDEX_DTYPES.get(expert_idx.dtype), _GATE_DTYPES.get(expert_weight.dtype)
    if (idx_code is None or gate_code is None or expert_idx.dim() != 2 or num_tokens == 0 or k == 0
            or not _layer_operands_ok(x, w1, w2) or not _valid_tokens_ok(valid_tokens)
            or expert_idx.device != x.device or expert_weight.device != x.device
            or not expert_idx.is_contiguous() or not expert_weight.is_contiguous()):
        return None
    size = layer_bytes(0, num_tokens * k, num_experts, d_model, ffn_dim)
    if size is None:
        return None
    dev = x.device
    workspace = torch.empty(size, dtype=torch.uint8, device=dev)
    out = torch.empty(num_tokens, d_model, dtype=torch.bfloat16, device=dev)
    check(lib().sb_layer(
        x.data_ptr(), expert_idx.data_ptr(), idx_code, expert_weight.data_ptr(), gate_code, w1.data_ptr(),
        w2.data_ptr(), out.data_ptr(), workspace.data_ptr(), size, num_tokens, k, num_experts, d_model, ffn_dim,
        _ptr(valid_tokens), stream_of(dev),
    ))
    return out


def layer_assigned_cuda(x: torch.Tensor, token_of_copy: torch.Tensor, expert_of_copy: torch.Tensor,
                        weight_of_copy: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor,
                        valid_tokens: torch.Tensor | None) -> torch.Tensor | None:
    """moe_forward_assigned's stages as one call, or None as in layer_cuda. The
    list's three tensors are 1-D, of one length, not empty."""
    num_experts, d_model, ffn_dim = w1.shape
    num_tokens, n = x.shape[0], expert_of_copy.numel()
    token_code, expert_code = _INDEX_DTYPES.get(token_of_copy.dtype), _INDEX_DTYPES.get(expert_of_copy.dtype)
    gate_code = _GATE_DTYPES.get(weight_of_copy.dtype)
    dev = x.device
    if (token_code is None or expert_code is None or gate_code is None or num_tokens == 0
            or not _layer_operands_ok(x, w1, w2) or not _valid_tokens_ok(valid_tokens)
            or token_of_copy.device != dev or expert_of_copy.device != dev or weight_of_copy.device != dev
            or not token_of_copy.is_contiguous() or not expert_of_copy.is_contiguous()
            or not weight_of_copy.is_contiguous()):
        return None
    size = layer_bytes(num_tokens, n, num_experts, d_model, ffn_dim)
    if size is None:
        return None
    workspace = torch.empty(size, dtype=torch.uint8, device=dev)
    out = torch.empty(num_tokens, d_model, dtype=torch.bfloat16, device=dev)
    check(lib().sb_layer_assigned(
        x.data_ptr(), token_of_copy.data_ptr(), token_code, expert_of_copy.data_ptr(), expert_code,
        weight_of_copy.data_ptr(), gate_code, w1.data_ptr(), w2.data_ptr(), out.data_ptr(), workspace.data_ptr(), size,
        n, num_tokens, num_experts, d_model, ffn_dim, _ptr(valid_tokens), stream_of(dev),
    ))
    return out


def layer_rounded_cuda(x: torch.Tensor, scores: torch.Tensor, k: int, w1: torch.Tensor, w2: torch.Tensor,
                       tile: int) -> torch.Tensor | None:
    """moe_forward_rounded's stages as one call, or None as in layer_cuda."""
    num_experts, d_model, ffn_dim = w1.shape
    num_tokens = x.shape[0]
    dev = x.device
    if (not _layer_operands_ok(x, w1, w2) or scores.device != dev or scores.dtype is not torch.float32
            or scores.dim() != 2 or not scores.is_contiguous() or num_tokens == 0):
        return None
    size = layer_rounded_bytes(num_tokens, num_experts, k, tile, d_model, ffn_dim)
    if size is None:
        return None
    workspace = torch.empty(size, dtype=torch.uint8, device=dev)
    out = torch.empty(num_tokens, d_model, dtype=torch.bfloat16, device=dev)
    check(lib().sb_layer_rounded(
        x.data_ptr(), scores.data_ptr(), w1.data_ptr(), w2.data_ptr(), out.data_ptr(), workspace.data_ptr(), size,
        num_tokens, num_experts, k, tile, d_model, ffn_dim, stream_of(dev),
    ))
    return out


# ---- the layer with gated experts, forward and backward (this build's C ABI) ----

_ACTIVATIONS = {"silu": 0, "gelu": 1}


_HERE = contextlib.nullcontext()


def _device_of(t: torch.Tensor) -> contextlib.AbstractContextManager:
    """Makes t's device current for a launch, where it is not."""
    return _HERE if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


@functools.lru_cache(maxsize=256)
def gated_bytes(num_tokens: int, k: int, num_experts: int, d_model: int, ffn_dim: int) -> tuple[int, int, int, int]:
    """Bytes of gated_layer_cuda's workspace, of what gated_train_cuda keeps, and of
    its and gated_backward_cuda's workspaces."""
    sizes = [ctypes.c_int64() for _ in range(4)]
    check(lib().sb_gated_sizes(num_tokens, k, num_experts, d_model, ffn_dim, *(ctypes.byref(s) for s in sizes)))
    return tuple(s.value for s in sizes)


def _check_gated(x: torch.Tensor, expert_idx: torch.Tensor | None, gates: torch.Tensor, w1: torch.Tensor,
                 w2: torch.Tensor, activation: str, valid_tokens: torch.Tensor | None) -> tuple[int, ...]:
    """(T, k, E, D, F) of operands that the gated layer's calls take as they are."""
    try:
        (num_tokens, d_model), (rows, k), (num_experts, ffn_dim, columns) = x.shape, gates.shape, w2.shape
    except ValueError:
        _fail(f"x must be [T, D], expert_weight [T, k], w1 [E, D, 2F] and w2 [E, F, D], got {_shape(x)}, {_shape(gates)}, "
              f"{_shape(w1)} and {_shape(w2)}")
    device = x.get_device()
    if (device < 0 or w1.get_device() != device or w2.get_device() != device or gates.get_device() != device
            or (expert_idx is not None and expert_idx.get_device() != device)):
        _fail("all inputs must be on the same GPU")
    if not (x.dtype is w1.dtype is w2.dtype is torch.bfloat16):
        _fail("x, w1 and w2 must be bfloat16")
    if columns != d_model or w1.shape != (num_experts, d_model, 2 * ffn_dim):
        _fail(f"x must be [T, D], w1 [E, D, 2F] and w2 [E, F, D], got {_shape(x)}, {_shape(w1)} and {_shape(w2)}")
    if not (x.is_contiguous() and w1.is_contiguous() and w2.is_contiguous()):
        _fail("x, w1 and w2 must be contiguous")
    if (x.data_ptr() | w1.data_ptr() | w2.data_ptr()) % 16:
        _fail("x, w1 and w2 must be 16-byte aligned")
    if rows != num_tokens or k == 0:
        _fail(f"expert_weight must be [T, k] with k > 0, got {_shape(gates)}")
    if gates.dtype not in _GATE_DTYPES:
        _fail(f"expert_weight must be bfloat16, float16 or float32, got {gates.dtype}")
    if expert_idx is not None:
        if expert_idx.shape != gates.shape:
            _fail(f"expert_idx must be [T, k] as expert_weight, got {_shape(expert_idx)}")
        if expert_idx.dtype not in _INDEX_DTYPES:
            _fail(f"expert_idx must be int32 or int64, got {expert_idx.dtype}")
    if not 0 < num_experts <= _MAX_EXPERTS:
        _fail(f"num_experts must be in [1, {_MAX_EXPERTS}], got {num_experts}")
    if activation not in _ACTIVATIONS:
        _fail(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if valid_tokens is not None and not (valid_tokens.get_device() == device and _valid_tokens_ok(valid_tokens)):
        _fail("valid_tokens must be a one-element int32 CUDA tensor")
    return num_tokens, k, num_experts, d_model, ffn_dim


def gated_layer_cuda(x: torch.Tensor, expert_idx: torch.Tensor, expert_weight: torch.Tensor, w1: torch.Tensor,
                     w2: torch.Tensor, activation: str, valid_tokens: torch.Tensor | None = None) -> torch.Tensor:
    """The layer with gated experts: out [T, D] bf16. Rows t >= valid_tokens (if given) are left unwritten."""
    t, k, e, d, f = _check_gated(x, expert_idx, expert_weight, w1, w2, activation, valid_tokens)
    out = torch.empty_like(x)
    if t == 0:
        return out
    expert_idx, gates = expert_idx.contiguous(), expert_weight.contiguous()
    size = gated_bytes(t, k, e, d, f)[0]
    workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
    with _device_of(x):
        check(lib().sb_gated_layer(
            x.data_ptr(), expert_idx.data_ptr(), _INDEX_DTYPES[expert_idx.dtype], gates.data_ptr(),
            _GATE_DTYPES[gates.dtype], w1.data_ptr(), w2.data_ptr(), out.data_ptr(), _ACTIVATIONS[activation],
            workspace.data_ptr(), size, t, k, e, d, f, _ptr(valid_tokens), stream_of(x.device),
        ))
    return out


def gated_train_cuda(x: torch.Tensor, expert_idx: torch.Tensor, expert_weight: torch.Tensor, w1: torch.Tensor,
                     w2: torch.Tensor, activation: str, valid_tokens: torch.Tensor | None = None
                     ) -> tuple[torch.Tensor, torch.Tensor]:
    """(out, saved): gated_layer_cuda's output, and the bytes that gated_backward_cuda reads."""
    t, k, e, d, f = _check_gated(x, expert_idx, expert_weight, w1, w2, activation, valid_tokens)
    out = torch.empty_like(x)
    if t == 0:
        return out, torch.empty(0, dtype=torch.uint8, device=x.device)
    expert_idx, gates = expert_idx.contiguous(), expert_weight.contiguous()
    _, saved_size, size, _ = gated_bytes(t, k, e, d, f)
    saved = torch.empty(saved_size, dtype=torch.uint8, device=x.device)
    workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
    with _device_of(x):
        check(lib().sb_gated_train(
            x.data_ptr(), expert_idx.data_ptr(), _INDEX_DTYPES[expert_idx.dtype], gates.data_ptr(),
            _GATE_DTYPES[gates.dtype], w1.data_ptr(), w2.data_ptr(), out.data_ptr(), _ACTIVATIONS[activation],
            saved.data_ptr(), saved_size, workspace.data_ptr(), size, t, k, e, d, f, _ptr(valid_tokens),
            stream_of(x.device),
        ))
    return out, saved


def gated_backward_cuda(grad_out: torch.Tensor, x: torch.Tensor, expert_weight: torch.Tensor, w1: torch.Tensor,
                        w2: torch.Tensor, saved: torch.Tensor, activation: str,
                        valid_tokens: torch.Tensor | None = None
                        ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients (x, expert_weight, w1, w2) of gated_train_cuda's output, each of its operand's shape and dtype.
    saved: what that call kept. Rows t >= valid_tokens (if given) of the first two are left unwritten."""
    t, k, e, d, f = _check_gated(x, None, expert_weight, w1, w2, activation, valid_tokens)
    if grad_out.device != x.device or grad_out.dtype != torch.bfloat16 or grad_out.shape != x.shape:
        _fail(f"grad_out must be a {_shape(x)} bfloat16 tensor on the same GPU, got {_shape(grad_out)} {grad_out.dtype}")
    if t == 0:
        return torch.empty_like(x), torch.empty_like(expert_weight), torch.zeros_like(w1), torch.zeros_like(w2)
    _, saved_size, _, size = gated_bytes(t, k, e, d, f)
    if not (saved.device == x.device and saved.dtype == torch.uint8 and saved.numel() == saved_size
            and saved.is_contiguous()):
        _fail("saved is not what gated_train_cuda kept for these operands")
    grad_out, gates = grad_out.contiguous(), expert_weight.contiguous()
    if grad_out.data_ptr() % 16:
        grad_out = grad_out.clone()
    grads = torch.empty_like(x), torch.empty_like(gates), torch.empty_like(w1), torch.empty_like(w2)
    workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
    with _device_of(x):
        check(lib().sb_gated_backward(
            grad_out.data_ptr(), x.data_ptr(), gates.data_ptr(), _GATE_DTYPES[gates.dtype], w1.data_ptr(),
            w2.data_ptr(), saved.data_ptr(), saved_size, *(g.data_ptr() for g in grads), _ACTIVATIONS[activation],
            workspace.data_ptr(), size, t, k, e, d, f, _ptr(valid_tokens), stream_of(x.device),
        ))
    return grads


# ---- the AdamW step (this build's C ABI) ----

QUANT_BLOCK = 256


_dtype_of, _shape_of = operator.attrgetter("dtype"), operator.attrgetter("shape")
_addresses = functools.partial(map, torch.Tensor.data_ptr)
_lengths = functools.partial(map, torch.Tensor.numel)


def _check_list(tensors, device: int, what: str, dtype: torch.dtype | None = None, lengths=None) -> None:
    """All contiguous, on GPU `device`, of one dtype and of these lengths, if given. (Whole
    lists at a time: a step of many small tensors is bound by these checks.)"""
    if not set(map(torch.Tensor.get_device, tensors)) <= {device}:
        _fail(f"{what} must be on the step's GPU")
    if not all(map(torch.Tensor.is_contiguous, tensors)):
        _fail(f"{what} must be contiguous")
    if dtype is not None and not set(map(_dtype_of, tensors)) <= {dtype}:
        _fail(f"{what} must be {dtype}")
    if lengths is not None and list(_lengths(tensors)) != lengths:
        _fail(f"{what} must have the parameters' lengths")


def _state_lists(states, eight: bool, signed: bool, name: str, device: int, lengths: list[int]):
    """(values or codes, scales or None) of a list of states, checked."""
    if any(isinstance(s, torch.Tensor) == eight for s in states):
        _fail("all states must be of one kind: float32 tensors, or 8-bit codes and scales")
    if not eight:
        _check_list(states, device, f"float32 states ({name})", torch.float32, lengths)
        return states, None
    codes, scales = [s[0] for s in states], [s[1] for s in states]
    _check_list(codes, device, f"{name} codes", torch.int8 if signed else torch.uint8, lengths)
    _check_list(scales, device, f"{name} scales (one for each {QUANT_BLOCK} values)", torch.float32,
                [-(-n // QUANT_BLOCK) for n in lengths])
    return codes, scales


def _device_scalar(t, name: str, device: torch.device) -> int | None:
    if not isinstance(t, torch.Tensor):
        return None
    if t.device != device or t.dtype != torch.float32 or t.numel() != 1:
        _fail(f"{name} must be a number or a one-element float32 tensor on the parameters' GPU")
    return t.data_ptr()


def adamw_cuda(params, grads, masters, exp_avgs, exp_avg_sqs, step: torch.Tensor, lr, beta1: float, beta2: float,
               eps: float, weight_decay: float, grad_scale, seed: int) -> None:
    """One AdamW step of a list of tensors, in place (include/sparsebench_hip.h: sb_adamw).

    exp_avgs / exp_avg_sqs: fp32 tensors, or (codes, scales) pairs of 8-bit
    states; masters: None or a list of fp32 tensors; step [2] int32."""
    n = len(params)
    if not (len(grads) == len(exp_avgs) == len(exp_avg_sqs) == n) or (masters is not None and len(masters) != n):
        _fail("params, grads, masters and states must be lists of one length")
    if not (step.is_cuda and step.dtype == torch.int32 and step.numel() == 2 and step.is_contiguous()):
        _fail("step must be a contiguous int32 CUDA tensor of two elements")
    dev, index = step.device, step.get_device()
    eight = n > 0 and not isinstance(exp_avgs[0], torch.Tensor)
    _check_list(params, index, "parameters")
    _check_list(grads, index, "gradients")
    if list(map(_shape_of, params)) != list(map(_shape_of, grads)):
        _fail("each gradient must have its parameter's shape")
    lengths = list(_lengths(params))
    if masters is not None:
        _check_list(masters, index, "masters", torch.float32, lengths)
    m, m_scales = _state_lists(exp_avgs, eight, True, "exp_avg", index, lengths)
    v, v_scales = _state_lists(exp_avg_sqs, eight, False, "exp_avg_sq", index, lengths)
    try:
        codes = [_GATE_DTYPES[p] | _GATE_DTYPES[g] << 32
                 for p, g in zip(map(_dtype_of, params), map(_dtype_of, grads))]
    except KeyError as e:
        _fail(f"parameters and gradients must be bfloat16, float16 or float32, got {e.args[0]}")
    none = itertools.repeat(0)
    words = array.array("q", itertools.chain.from_iterable(zip(
        _addresses(params), _addresses(grads), none if masters is None else _addresses(masters), _addresses(m),
        _addresses(v), _addresses(m_scales) if eight else none, _addresses(v_scales) if eight else none, lengths,
        codes)))
    lr_ptr, scale_ptr = _device_scalar(lr, "lr", dev), _device_scalar(grad_scale, "grad_scale", dev)
    with _device_of(step):
        if scale_ptr is None and grad_scale is not None:  # a number: as a device scalar
            scale = torch.full((1,), float(grad_scale), dtype=torch.float32, device=dev)
            scale_ptr = scale.data_ptr()
        check(lib().sb_adamw(words.buffer_info()[0], n, 8 if eight else 32, step.data_ptr(),
                             0.0 if lr_ptr else float(lr), lr_ptr, beta1, beta2, eps, weight_decay, scale_ptr,
                             seed & 0xFFFFFFFF, stream_of(dev)))
    # Written through their addresses: a graph that saved one of them has to be told (0.05 us a tensor).
    torch.autograd.graph.increment_version([*params, *(masters or ())])


def dequantize_cuda(pairs, dtype: torch.dtype) -> list[torch.Tensor]:
    """The values of 8-bit states, (codes, scales) each, in `dtype` (include/sparsebench_hip.h: sb_dequantize)."""
    if dtype not in _GATE_DTYPES:
        _fail(f"values must be bfloat16, float16 or float32, got {dtype}")
    if not pairs:
        return []
    all_codes, all_scales = [p[0] for p in pairs], [p[1] for p in pairs]
    dev = all_codes[0].device
    if dev.type != "cuda":
        _fail("codes must be CUDA tensors")
    lengths = list(_lengths(all_codes))
    _check_list(all_codes, dev.index, "codes")
    _check_list(all_scales, dev.index, f"scales (one for each {QUANT_BLOCK} values)", torch.float32,
                [-(-n // QUANT_BLOCK) for n in lengths])
    dtypes = list(map(_dtype_of, all_codes))
    if not set(dtypes) <= {torch.int8, torch.uint8}:
        _fail(f"codes must be int8 or uint8, got {set(dtypes)}")
    # Each value list starts at a multiple of 16 bytes of one buffer, which is
    # cut into value lists and the gaps after them by one call.
    step = 16 // dtype.itemsize
    gaps = [-n % step for n in lengths]
    flat = torch.empty(sum(lengths) + sum(gaps), dtype=dtype, device=dev)
    pieces = flat.split_with_sizes(list(itertools.chain.from_iterable(zip(lengths, gaps))))[::2]
    out = [o if codes.dim() == 1 else o.view(codes.shape) for o, codes in zip(pieces, all_codes)]
    words = array.array("q", itertools.chain.from_iterable(zip(
        _addresses(all_codes), _addresses(all_scales), _addresses(out), lengths,
        [1 if d == torch.int8 else 0 for d in dtypes])))
    with _device_of(flat):
        check(lib().sb_dequantize(words.buffer_info()[0], len(pairs), _GATE_DTYPES[dtype], stream_of(dev)))
    return out


# ---- norms before and after a block (this build's C ABI) ----

_NORM_MAX_D = 32768


def _check_rows(t: torch.Tensor, name: str, like: torch.Tensor | None = None) -> None:
    """[T, D] with contiguous rows on a GPU; with `like`, of its shape, type and device."""
    shape = t.shape
    if t.get_device() < 0 or len(shape) != 2 or t.dtype not in _GATE_DTYPES:
        _fail(f"{name} must be a [T, D] bfloat16, float16 or float32 CUDA tensor, got {_shape(t)} {t.dtype}")
    if like is not None and (shape != like.shape or t.dtype is not like.dtype or t.get_device() != like.get_device()):
        _fail(f"{name} must be a {_shape(like)} {like.dtype} tensor on {like.device}, got {_shape(t)} {t.dtype} on "
              f"{t.device}")
    if not t.is_contiguous() and shape[1] != 1 and t.stride(1) != 1:
        _fail(f"{name} must have contiguous rows")
    if not 0 < shape[1] <= _NORM_MAX_D:
        _fail(f"rows must have 1 to {_NORM_MAX_D} values, got {shape[1]}")


def _new_rows(like: torch.Tensor) -> torch.Tensor:
    """Contiguous, of like's shape and type (empty_like takes half of empty's 1.9 us, but keeps strides)."""
    return torch.empty_like(like) if like.is_contiguous() else torch.empty(like.shape, dtype=like.dtype, device=like.device)


def _check_vector(t: torch.Tensor | None, name: str, like: torch.Tensor) -> int:
    """Its dtype's code."""
    if t is None:
        return 0
    code = _GATE_DTYPES.get(t.dtype)
    if code is None or t.get_device() != like.get_device() or t.shape != like.shape[1:] or not t.is_contiguous():
        _fail(f"{name} must be a contiguous [{like.shape[1]}] bfloat16, float16 or float32 tensor on {like.device}")
    return code


def _check_norm_gate(gate: torch.Tensor | None, like: torch.Tensor) -> tuple[int, int, int]:
    """(dtype's code, kind, row stride) of a gate."""
    if gate is None:
        return 0, 0, 0
    t, d = like.shape
    code = _GATE_DTYPES.get(gate.dtype)
    if code is None or gate.get_device() != like.get_device():
        _fail(f"gate must be a bfloat16, float16 or float32 tensor on {like.device}, got {gate.dtype} on {gate.device}")
    if gate.shape == (d,) and gate.is_contiguous():
        return code, 1, 0
    if gate.shape == (t, d) and (d == 1 or gate.stride(1) == 1):
        return code, 3, gate.stride(0)
    if gate.shape == (t, 1):
        return code, 2, gate.stride(0)
    _fail(f"gate must be [D], [T, 1] or [T, D] with contiguous rows, got {_shape(gate)}")


def _check_norm(eps: float, valid_tokens: torch.Tensor | None, like: torch.Tensor) -> None:
    if not eps >= 0:
        _fail(f"eps must not be negative, got {eps}")
    if valid_tokens is not None and not (valid_tokens.get_device() == like.get_device() and _valid_tokens_ok(valid_tokens)):
        _fail("valid_tokens must be a one-element int32 CUDA tensor")


def norm_in_cuda(x: torch.Tensor, weight: torch.Tensor | None, eps: float,
                 valid_tokens: torch.Tensor | None = None) -> torch.Tensor:
    """weight x / sqrt(mean(x^2) + eps) of each row (include/sparsebench_hip.h: sb_norm_in)."""
    _check_rows(x, "x")
    weight_code = _check_vector(weight, "weight", x)
    _check_norm(eps, valid_tokens, x)
    out = _new_rows(x)
    with _device_of(x):
        check(lib().sb_norm_in(x.data_ptr(), x.stride(0), _ptr(weight), weight_code, out.data_ptr(),
                               _GATE_DTYPES[x.dtype], *x.shape, eps, _ptr(valid_tokens), stream_of(x.device)))
    return out


def norm_out_cuda(y: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, gate: torch.Tensor | None,
                  scale: float, eps: float, next_weight: torch.Tensor | None,
                  valid_tokens: torch.Tensor | None = None):
    """x + scale gate weight n(y), or that and its own norm (sb_norm_out)."""
    _check_rows(x, "x")
    _check_rows(y, "y", x)
    weight_code, next_code = _check_vector(weight, "weight", x), _check_vector(next_weight, "next_weight", x)
    gate_code, kind, gate_stride = _check_norm_gate(gate, x)
    _check_norm(eps, valid_tokens, x)
    out = _new_rows(x)
    following = None if next_weight is None else torch.empty_like(out)
    with _device_of(x):
        check(lib().sb_norm_out(
            y.data_ptr(), y.stride(0), x.data_ptr(), x.stride(0), _ptr(weight), weight_code, _ptr(gate),
            gate_code, kind, gate_stride, scale, _ptr(next_weight), next_code, out.data_ptr(),
            _ptr(following), _GATE_DTYPES[x.dtype], *x.shape, eps, _ptr(valid_tokens), stream_of(x.device)))
    return out if following is None else (out, following)


@functools.lru_cache(maxsize=256)
def _norm_bytes(num_tokens: int, d_model: int, device: int) -> int:
    size = ctypes.c_int64()
    check(lib().sb_norm_sizes(num_tokens, d_model, ctypes.byref(size)))
    return size.value


def _norm_workspace(like: torch.Tensor) -> torch.Tensor:
    """For the device that is current, like's."""
    return torch.empty(_norm_bytes(*like.shape, like.get_device()), dtype=torch.uint8, device=like.device)


def norm_in_backward_cuda(grad: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, eps: float,
                          grad_x: torch.Tensor | None, valid_tokens: torch.Tensor | None = None
                          ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The gradients (x, weight) of norm_in_cuda, x's with grad_x added (sb_norm_in_backward)."""
    _check_rows(x, "x")
    _check_rows(grad, "grad", x)
    if grad_x is not None:
        _check_rows(grad_x, "grad_x", x)
    weight_code = _check_vector(weight, "weight", x)
    _check_norm(eps, valid_tokens, x)
    dx = _new_rows(x)
    if x.shape[0] == 0:  # sums of nothing
        return dx, None if weight is None else torch.zeros_like(weight)
    dweight = None if weight is None else torch.empty_like(weight)
    with _device_of(x):
        workspace = _norm_workspace(x)
        check(lib().sb_norm_in_backward(
            grad.data_ptr(), grad.stride(0), x.data_ptr(), x.stride(0), _ptr(weight), weight_code,
            _ptr(grad_x), 0 if grad_x is None else grad_x.stride(0), dx.data_ptr(), _ptr(dweight),
            _GATE_DTYPES[x.dtype], *x.shape, eps, _ptr(valid_tokens), workspace.data_ptr(), workspace.numel(),
            stream_of(x.device)))
    return dx, dweight


def norm_out_backward_cuda(grad_out: torch.Tensor, y: torch.Tensor, weight: torch.Tensor | None,
                           gate: torch.Tensor | None, scale: float, eps: float, out: torch.Tensor | None,
                           grad_next: torch.Tensor | None, next_weight: torch.Tensor | None,
                           valid_tokens: torch.Tensor | None = None):
    """The gradients (y, x, weight, gate, next_weight) of norm_out_cuda (sb_norm_out_backward)."""
    _check_rows(y, "y")
    _check_rows(grad_out, "grad_out", y)
    if (grad_next is None) != (next_weight is None) or (grad_next is not None and out is None):
        _fail("the next norm's gradient needs grad_next, next_weight and out")
    if grad_next is not None:
        _check_rows(grad_next, "grad_next", y)
        _check_rows(out, "out", y)
    weight_code, next_code = _check_vector(weight, "weight", y), _check_vector(next_weight, "next_weight", y)
    gate_code, kind, gate_stride = _check_norm_gate(gate, y)
    _check_norm(eps, valid_tokens, y)
    if y.shape[0] == 0:  # sums of nothing
        return (torch.empty_like(y), grad_out, *(None if w is None else torch.zeros_like(w)
                                                 for w in (weight, gate, next_weight)))
    dy = _new_rows(y)
    dx = None if grad_next is None else _new_rows(y)
    dweight, dnext = (None if w is None else torch.empty_like(w) for w in (weight, next_weight))
    dgate = None if gate is None else torch.empty(gate.shape, dtype=gate.dtype, device=gate.device)
    following = out if grad_next is not None else None
    with _device_of(y):
        workspace = _norm_workspace(y)
        check(lib().sb_norm_out_backward(
            grad_out.data_ptr(), grad_out.stride(0), _ptr(grad_next), 0 if grad_next is None else grad_next.stride(0),
            y.data_ptr(), y.stride(0), _ptr(following), 0 if following is None else following.stride(0),
            _ptr(weight), weight_code, _ptr(gate), gate_code, kind, gate_stride, scale, _ptr(next_weight), next_code,
            dy.data_ptr(), _ptr(dx), _ptr(dweight), _ptr(dgate),
            _ptr(dnext), _GATE_DTYPES[y.dtype], *y.shape, eps, _ptr(valid_tokens), workspace.data_ptr(),
            workspace.numel(), stream_of(y.device)))
    return dy, grad_out if dx is None else dx, dweight, dgate, dnext


# ---- gated experts with 4-bit weights (this build's C ABI) ----

_MAX_COPIES4 = 2048


@functools.lru_cache(maxsize=256)
def _experts4_bytes(num_tokens: int, k: int, num_experts: int, d_model: int, ffn_dim: int, device: int) -> int:
    size = ctypes.c_int64()
    check(lib().sb_experts4_sizes(num_tokens, k, num_experts, d_model, ffn_dim, ctypes.byref(size)))
    return size.value


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(E, K, N) of 4-bit weights."""
    shape = codes.shape
    if (len(shape) != 5 or shape[3] != 32 or shape[4] != 16 or scales.shape != shape[:4] or codes.get_device() < 0
            or codes.get_device() != scales.get_device() or not codes.dtype is scales.dtype is torch.uint8):
        _fail(f"{name} must be uint8 codes [E, N/32, K/32, 32, 16] and scales [E, N/32, K/32, 32] on one GPU, got "
              f"{_shape(codes)} {codes.dtype} and {_shape(scales)} {scales.dtype}")
    if not (codes.is_contiguous() and scales.is_contiguous()) or codes.data_ptr() % 16:
        _fail(f"{name} must be contiguous, its codes 16-byte aligned")
    return shape[0], 32 * shape[2], 32 * shape[1]


def experts4_layer_cuda(x: torch.Tensor, expert_idx: torch.Tensor, expert_weight: torch.Tensor, w1, w2,
                        activation: str, valid_tokens: torch.Tensor | None = None) -> torch.Tensor:
    """gated_layer_cuda with (codes, scales) pairs as weights (include/sparsebench_hip.h: sb_experts4_layer)."""
    (c1, s1), (c2, s2) = w1, w2
    try:
        (t, width), (rows, k) = x.shape, expert_idx.shape
    except ValueError:
        t, width, rows, k = 0, 0, -1, 0
    if t != rows or expert_idx.shape != expert_weight.shape:
        _fail(f"x must be [T, D], expert_idx and expert_weight [T, k], got {_shape(x)}, {_shape(expert_idx)} and "
              f"{_shape(expert_weight)}")
    (e, d, columns), (experts, f, out_columns) = _check_codes(c1, s1, "w1"), _check_codes(c2, s2, "w2")
    if e != experts or width != d or out_columns != d or columns != 2 * f:
        _fail(f"x must be [T, D], w1 of [E, D, 2F] and w2 of [E, F, D], got {_shape(x)}, {[e, d, columns]} and "
              f"{[experts, f, out_columns]}")
    device = x.get_device()
    if not (device == expert_idx.get_device() == expert_weight.get_device() == c1.get_device() == c2.get_device()):
        _fail("all inputs must be on the same GPU")
    if x.dtype is not torch.bfloat16 or not x.is_contiguous() or x.data_ptr() % 16:
        _fail("x must be contiguous 16-byte aligned bfloat16")
    gate_code, index_code = _GATE_DTYPES.get(expert_weight.dtype), _INDEX_DTYPES.get(expert_idx.dtype)
    if gate_code is None:
        _fail(f"expert_weight must be bfloat16, float16 or float32, got {expert_weight.dtype}")
    if index_code is None:
        _fail(f"expert_idx must be int32 or int64, got {expert_idx.dtype}")
    if activation not in _ACTIVATIONS:
        _fail(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if valid_tokens is not None and not (valid_tokens.get_device() == device and _valid_tokens_ok(valid_tokens)):
        _fail("valid_tokens must be a one-element int32 CUDA tensor")
    if k == 0:
        _fail(f"expert_weight must be [T, k] with k > 0, got {_shape(expert_weight)}")
    if t * k > _MAX_COPIES4:
        _fail(f"at most {_MAX_COPIES4} copies (T k), got {t * k}: more are faster through dequantize_experts and "
              "moe_forward_gated")
    out = torch.empty_like(x)
    if t == 0:
        return out
    expert_idx, gates = expert_idx.contiguous(), expert_weight.contiguous()
    with _device_of(x):
        size = _experts4_bytes(t, k, e, d, f, device)
        workspace = torch.empty(size, dtype=torch.uint8, device=x.device)
        check(lib().sb_experts4_layer(
            x.data_ptr(), expert_idx.data_ptr(), index_code, gates.data_ptr(), gate_code, c1.data_ptr(), s1.data_ptr(),
            c2.data_ptr(), s2.data_ptr(), out.data_ptr(), _ACTIVATIONS[activation], workspace.data_ptr(), size, t, k, e,
            d, f, _ptr(valid_tokens), stream_of(x.device)))
    return out


def quantize4_cuda(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of w [E, K, N] (include/sparsebench_hip.h: sb_quantize4)."""
    if not w.is_cuda or w.dim() != 3 or w.dtype not in _GATE_DTYPES:
        _fail(f"w must be an [E, K, N] bfloat16, float16 or float32 CUDA tensor, got {_shape(w)} {w.dtype}")
    e, k, n = w.shape
    if e == 0 or k == 0 or n == 0 or k % 32 or n % 32:
        _fail(f"K and N must be positive multiples of 32, got {_shape(w)}")
    w = w.contiguous()
    scales = torch.empty(e, n // 32, k // 32, 32, dtype=torch.uint8, device=w.device)
    codes = torch.empty(*scales.shape, 16, dtype=torch.uint8, device=w.device)
    with _device_of(w):
        check(lib().sb_quantize4(w.data_ptr(), _GATE_DTYPES[w.dtype], codes.data_ptr(), scales.data_ptr(), e, k, n,
                                 stream_of(w.device)))
    return codes, scales


def dequantize4_cuda(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """w [E, K, N] bf16 of codes and scales (include/sparsebench_hip.h: sb_dequantize4)."""
    e, k, n = _check_codes(codes, scales, "w")
    w = torch.empty(e, k, n, dtype=torch.bfloat16, device=codes.device)
    if w.numel():
        with _device_of(codes):
            check(lib().sb_dequantize4(codes.data_ptr(), scales.data_ptr(), w.data_ptr(), e, k, n,
                                       stream_of(codes.device)))
    return w


# ---- orthogonalised updates (this build's C ABI) ----

_MAX_STEPS = 32


def _stack_of(t: torch.Tensor, what: str, written: bool) -> tuple[int, int, int, int, int]:
    """(matrices, rows, columns, stride of matrices, of rows) of a tensor [..., rows, columns]
    whose rows are contiguous and whose leading dimensions are one; of tensors that are
    written, no two elements in one place."""
    if t.dim() < 2:
        _fail(f"{what} must be matrices [..., rows, columns], got {_shape(t)}")
    rows, columns = t.shape[-2:]
    if columns > 1 and t.stride(-1) != 1:
        _fail(f"{what} must have contiguous rows")
    matrices, stride = 1, 0
    for size, step in zip(reversed(t.shape[:-2]), reversed(t.stride()[:-2])):
        if size == 1:
            continue
        if matrices > 1 and step != matrices * stride:
            _fail(f"{what} must have leading dimensions that are one stride apart")
        stride = step if matrices == 1 else stride
        matrices *= size
    if written and t.numel() > 0:
        span = 1
        for size, step in sorted(((s, d) for s, d in ((matrices, stride), (rows, t.stride(-2)), (columns, 1)) if s > 1),
                                 key=lambda d: d[1]):
            if step < span:
                _fail(f"{what} must not overlap themselves")
            span += (size - 1) * step
    return matrices, rows, columns, stride, t.stride(-2)


def _check_stacks(tensors, device: int, what: str, dtypes, shapes=None) -> None:
    if not all(t.get_device() == device for t in tensors):
        _fail(f"{what} must be on one GPU")
    if not all(t.dtype in dtypes for t in tensors):
        _fail(f"{what} must be of {', '.join(str(d).removeprefix('torch.') for d in dtypes)}")
    if shapes is not None and list(map(_shape_of, tensors)) != shapes:
        _fail(f"{what} must have the parameters' shapes")


def _muon_words(params, grads, momenta, masters) -> array.array:
    """The list as sb_muon takes it (SbMuonTensor, 16 words each)."""
    words = array.array("q")
    none = itertools.repeat(None)
    for p, g, m, w in zip(params, grads, momenta or none, masters or none):
        stack = _stack_of(p, "parameters", True)
        _, _, _, *g_strides = _stack_of(g, "gradients", False)
        _, _, _, *m_strides = (0,) * 5 if m is None else _stack_of(m, "momenta", True)
        _, _, _, *w_strides = (0,) * 5 if w is None else _stack_of(w, "masters", True)
        words.extend((p.data_ptr(), g.data_ptr(), 0 if m is None else m.data_ptr(), 0 if w is None else w.data_ptr(),
                      *stack, *g_strides, *m_strides, *w_strides,
                      _GATE_DTYPES[p.dtype] | _GATE_DTYPES[g.dtype] << 32))
    return words


def _muon_workspace(words: array.array, count: int, device: torch.device) -> torch.Tensor:
    size = ctypes.c_int64()
    check(lib().sb_muon_sizes(words.buffer_info()[0], count, ctypes.byref(size)))
    return torch.empty(size.value, dtype=torch.uint8, device=device)


def _check_steps(steps: int) -> None:
    if not 1 <= steps <= _MAX_STEPS:
        _fail(f"steps must be 1 to {_MAX_STEPS}, got {steps}")


def muon_cuda(params, grads, momenta, masters, lr, momentum: float, nesterov: bool, weight_decay: float,
              update_rms: float, steps: int, grad_scale) -> None:
    """One orthogonalised step of a list of stacks of matrices, in place (include/sparsebench_hip.h: sb_muon)."""
    n = len(params)
    if not (len(grads) == len(momenta) == n) or (masters is not None and len(masters) != n):
        _fail("params, grads, momenta and masters must be lists of one length")
    _check_steps(steps)
    if not 0 <= momentum < 1:
        _fail(f"momentum must be in [0, 1), got {momentum}")
    if n == 0:
        return
    dev, index = params[0].device, params[0].get_device()
    if index < 0:
        _fail("parameters must be on one GPU")
    shapes = list(map(_shape_of, params))
    _check_stacks(params, index, "parameters", _GATE_DTYPES)
    _check_stacks(grads, index, "gradients", _GATE_DTYPES, shapes)
    _check_stacks(momenta, index, "momenta", (torch.float32,), shapes)
    if masters is not None:
        _check_stacks(masters, index, "masters", (torch.float32,), shapes)
    words = _muon_words(params, grads, momenta, masters)
    lr_ptr, scale_ptr = _device_scalar(lr, "lr", dev), _device_scalar(grad_scale, "grad_scale", dev)
    with _device_of(params[0]):
        if scale_ptr is None and grad_scale is not None:  # a number: as a device scalar
            scale = torch.full((1,), float(grad_scale), dtype=torch.float32, device=dev)
            scale_ptr = scale.data_ptr()
        workspace = _muon_workspace(words, n, dev)
        check(lib().sb_muon(words.buffer_info()[0], n, 0.0 if lr_ptr else float(lr), lr_ptr, momentum, int(nesterov),
                            weight_decay, update_rms, steps, scale_ptr, workspace.data_ptr(), workspace.numel(),
                            stream_of(dev)))
    torch.autograd.graph.increment_version([*params, *(masters or ())])


def orthogonalize_cuda(matrices: torch.Tensor, steps: int) -> torch.Tensor:
    """Newton-Schulz products of each matrix (include/sparsebench_hip.h: sb_orthogonalize)."""
    _check_steps(steps)
    if not matrices.is_cuda or matrices.dtype not in _GATE_DTYPES:
        _fail(f"matrices must be a bfloat16, float16 or float32 CUDA tensor, got {matrices.dtype} on {matrices.device}")
    out = torch.empty(matrices.shape, dtype=matrices.dtype, device=matrices.device)
    words = _muon_words([out], [matrices], None, None)
    with _device_of(matrices):
        workspace = _muon_workspace(words, 1, matrices.device)
        check(lib().sb_orthogonalize(words.buffer_info()[0], 1, steps, workspace.data_ptr(), workspace.numel(),
                                     stream_of(matrices.device)))
    return out
