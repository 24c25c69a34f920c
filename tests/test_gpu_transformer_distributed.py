"""The residual sums' gradient sinks under the reducer, and FusedMuon behind it: ranks that share the GPU."""
import pytest

pytestmark = pytest.mark.gpu


def test_muon_and_fused_residual_sums_under_ddp_sharing_the_gpu(tmp_path):
    """Kernels write the sums of norms and gates into the buckets, the C++ reducer sends them off when they are complete.  The
    attention core rounds its operands to 11 bits, so a different order of additions in front of it shows up as single
    roundings of 2^-11: 2e-3 of a gradient's norm, as for the other whole models."""
    import _muon_dist_workers as W
    from distributed_pytorch_amd import amp
    from test_gpu_distributed import _spawn_shared

    print("2 ranks on one device", flush=True)
    _spawn_shared(W.train, 2, (str(tmp_path), "native", "cuda"))
    amp.state().reset()
    W.check(str(tmp_path), 2, "cuda", 2e-3)
