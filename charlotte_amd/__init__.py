"""charlotte_amd — the quantized GGUF matrix product of plainsight-systems/charlotte
(Q4_0 and repacked Q6_K weights times f32 activations; decode GEMV and prefill
GEMM) as hand-written HIP for MI355X, behind the C ABI of
include/charlotte_hip_matmul.h. ``charlotte_amd.matmul`` is the operator
interface; ``charlotte_amd.serving`` what runs between a decoder step's products
and after its head (head norms and rotation, the quantized cache, attention,
probabilities, verification of drafted tokens); ``charlotte_amd.harness`` the device plumbing tests and the
benchmark use; ``charlotte_amd.synthetic`` the seeded inputs of the
benchmark's configurations.
"""

__all__ = ["matmul", "serving", "harness", "synthetic"]
