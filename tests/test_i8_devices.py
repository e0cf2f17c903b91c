"""The Python calls of the int8 rows and the sampler take operands of one GPU only: a host address
must not reach a kernel."""
import pytest
import torch

import libr3d_amd as R


def test_host_tensors_are_refused():
    x, q, s = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)
    for f in (lambda: R.quant_act_i8(x, q, s, n=8), lambda: R.gated_quant_i8(torch.cat((x, x), 1), q, s, n=8),
              lambda: R.rmsnorm_quant_i8(x, None, x[0], q, s, n=8),
              lambda: R.gemm_nt_q(q, s, q, s, torch.zeros(2, 2, dtype=torch.bfloat16), dtype="i8a8", N=2, K=8),
              lambda: R.sample_logits(torch.zeros(2, 8), s, torch.zeros(2, dtype=torch.int32), n_vocab=8)):
        with pytest.raises(ValueError, match="one GPU"):
            f()


@pytest.mark.gpu
def test_one_host_tensor_among_the_gpu_s(gpu):
    x, q, s = (torch.zeros(2, 8, dtype=t, device=gpu) for t in (torch.bfloat16, torch.int8, torch.float32))
    with pytest.raises(ValueError, match="one GPU"):
        R.quant_act_i8(x, q, s[:, 0].cpu(), n=8)
    with pytest.raises(ValueError, match="one GPU"):
        R.sample_logits(torch.zeros(2, 8, device=gpu), s[:, 0], torch.zeros(2, dtype=torch.int32, device=gpu), n_vocab=8,
                        top_k=torch.ones(2, dtype=torch.int32))
    assert R.quant_act_i8(x, q, s[:, 0].contiguous(), n=8) == R.RAD_OK
    torch.cuda.synchronize()
