"""gcnasm_amd -- block-scaled FP8 GEMM library for MI355X (gfx950).

The product is libgcnasm_amd.so (C ABI in include/gcnasm_amd.h): hand-written
HIP kernels for the MXFP8/MXFP4, DeepSeek block-scale and per-tensor FP8
GEMMs, the bf16 split-K GEMM with its graph-safe workspace handle, the
quantisers and layout shuffles that feed them, and the host launch logic
(tile manifest, heuristic, split-K geometry, kernarg blocks).

Python modules:
  f4gemm     mirror of the reference's f4gemm host namespace (MXFP8 path)
  opus_gemm  mirror of the reference's opus_gemm drivers (fp32-scale paths)
  flatmm_splitk  mirror of the reference's a16w16 split-K driver, workspace
             handle and split-K reduce
  mx4_cache  a key/value cache in MXFP4: append, attention over it, the weights of
             its tokens, eviction
  experts    layers of experts: the choice of each token's experts, the map of rows, each
             expert's rows times its weights in block scale, activation and weighted sum
  ops        tensor-level conveniences (torch tensors as device buffers)
"""
from ._lib import GaError, lib  # noqa: F401

__all__ = ["GaError", "lib"]
