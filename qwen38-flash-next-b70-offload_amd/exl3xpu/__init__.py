"""exl3xpu: EXL3 routed-expert offload for MI355X (HIP kernels behind the reference's exl3xpu_moe op schemas).

moe_offload  -- ops() loader, planar4 / pack_expert, ExpertStore (HBM slot cache + pinned host arena)
nvtier       -- TierStore, NvTier / NvTierFast / NvTierAsync (RAM tier with admission control)
routing      -- Router: logits to the picks and weights that the expert calls take
linear       -- FusedGroup: the dense EXL3 linear
fp8          -- Fp8Linear, Fp8Mlp: linears in 8-bit floats with a scale per 128 x 128 block
fp4          -- Fp4Linear, Fp4Mlp: linears in microscaled 4-bit floats
norm         -- RmsNorm: the norm before a layer's linears, with the residual's addition and quantised outputs
capi         -- ctypes binding of the C-ABI library libexl3moe.so (include/exl3moe.h)
synth        -- seeded synthetic experts and routing traces
"""
