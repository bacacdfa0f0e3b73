"""Static INT8 KV cache for vLLM on MI355X (gfx950): drop-in for the reference's `kvq` package.

  kvq.cuda_kernels   operator API (same names as the reference), HIP kernels via a C ABI
  kvq.block_cache    the INT8 cache with scales made as it is written (one per block of positions and head)
  kvq.scales         static-scale safetensors format: load / save / shard / merge_tp / for_layer
  kvq.synth          seeded synthetic workloads of the benchmark configurations
"""
