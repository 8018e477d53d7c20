"""MI355X-native MegaBlocks-style MoE forward path (routing -> SDD+GELU -> DSD -> combine).

A drop-in for the reference's sparsebench package on this path:
`sparsebench_amd.moe.moe_forward`, `sparsebench_amd.routing.route_device`,
`sparsebench_amd.spmm.sdd` / `dsd` and `sparsebench_amd._C` keep the
reference's names, arguments and results. The compute runs in hand-written
gfx950 HIP kernels of libsparsebench_hip.so, called through its C ABI.

Beside it, not in the reference: the layer with gated experts and its backward
pass (`moe.moe_forward_gated`, `moe_gated_train`, `moe_gated_backward`), the same
layer with 4-bit weights (`moe.moe_forward_gated_4bit`), the norms before and after
it (`norm`, `moe.moe_block_gated`), and the AdamW and orthogonalised steps of its
weights (`optim`).

The HIP library is loaded lazily (first op call), so the pure-Python parts
import on machines without a GPU.
"""
