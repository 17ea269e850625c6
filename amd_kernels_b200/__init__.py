"""B200-native kernels behind the amd_kernels entry points. The MXFP4 MoE layer is provided, and what
stands between two of them: ``amd_kernels_b200.moe.mxfp4_h6144_i768_e128_top4`` mirrors
``amd_kernels.moe.mxfp4_h6144_i768_e128_top4`` and adds ``add_rmsnorm_mxfp8``, ``LinearWeights``, ``mxfp8_linear`` and ``mxfp8_quant``."""
