"""HIP (gfx950) kernels of the TurboQuant packed-KV hot path.

Modules keep the reference's names (turboquant/kernels/__init__.py):
  packed_compress   bit-level helpers (sign permutation, unpacking) and the kernel-file codebook
  packed_attention  packed_attention: split-K decode over contiguous per-head packed arrays
  sparse_v          paged 3-bit decode over the reference's slot layout, dense and Sparse-V
  paged             paged packed cache: fused compression and GQA split-K decode
  paged8            paged cache of 8 bits a value: quantisation, decode and prefill attention
  evict8            accumulated attention weights over that cache, eviction of the tokens that got least
  plan              block tables, slots and positions of an engine step from the requests' lengths
  rotation          Walsh-Hadamard rotation of query / output rows, rotary positions on query / key rows
"""
