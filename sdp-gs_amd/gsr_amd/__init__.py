"""gsr_amd: host-side support of the MI355X Gaussian rasterizer (libgsr.so).

  _lib       ctypes binding of include/gsr.h (no CPU fallback)
  camera     reference camera maths (getWorld2View2 / getProjectionMatrix / focal2fov)
  synthetic  the seeded synthetic scenes of SURVEY.md 8(d)
  parallel   camera-sharded data parallelism with a bucketed RCCL all-reduce
  optim      fused Adam, global gradient norm and clipping
  linear     fused linear layer and gated pair (matrix products with their epilogues)
  feature_head  the head from the rendered 3-channel feature to wide features
"""
