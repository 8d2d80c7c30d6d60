"""exl3rocm -- MI355X-native EXL3 quantized-linear engine (drop-in for the reference plugin's
linear path).  Submodules:

  ops      torch custom ops exl3rocm::linear / exl3rocm::linear_groups
  paged    the attention step over a paged cache: batch_plan, rope_kv_write, paged_attention
  paged8   the same over a cache held in 8 bits: rope_kv_write8, kv_read8, paged_attention8
  plugin   Exl3Config / Exl3LinearMethod (vLLM quantization surface)
  kernels  tensor wrappers of the C ABI (reference extension call names)
  layout   safetensors checkpoint layout discovery
  synth    seeded synthetic layers (counter RNG)
"""
__all__ = ["ops", "paged", "paged8", "plugin", "kernels", "layout", "synth"]
