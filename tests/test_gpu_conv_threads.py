"""Two host threads that share a stream: convolutions whose launches hand copies of rows or weights over in a buffer of the stream do
not come between each other's."""
import numpy as np
import pytest
import torch

from fgms_amd import clouds
from tests import gpu_util as G
from tests.test_gpu_attention_threads import ROUNDS, both

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("channels", [64, 48])      # 48: over copies of the rows in channels of the tile
@pytest.mark.parametrize("dtype", [np.float16, np.float32], ids=["fp16", "fp32"])
def test_layers(dtype, channels):
    from fgms_amd import capi
    capi.set_kernel_policy(0)
    layers, plans, want, got = [], [], [], []
    for i in range(2):
        vox = clouds.cloud_indoor(clouds.rng_for(2), target=5000 + 1000 * i)
        D = G.to_dev(clouds.submanifold_case(vox, channels, channels, dtype, np.random.default_rng(i)))
        plans.append(capi.Plan(D["kpos"], D["imap"], D["omap"], D["n_in"], D["n_out"]))
        out = torch.empty(D["n_out"], channels, dtype=D["in_feats"].dtype, device="cuda")
        capi.conv_fwd(D["in_feats"], D["kernel"], out, D["kpos"], D["imap"], D["omap"], plan=plans[i])
        layers.append(D)
        want.append(out)
        got.append([torch.empty_like(out) for _ in range(ROUNDS)])
    count = [0, 0]
    torch.cuda.synchronize()

    def work(i):
        D = layers[i]
        capi.conv_fwd(D["in_feats"], D["kernel"], got[i][count[i]], D["kpos"], D["imap"], D["omap"], plan=plans[i])
        count[i] += 1

    both(work)
    mode = G.mode_of(dtype)
    for i in range(2):
        for t in got[i]:
            G.assert_close(t.cpu().numpy(), want[i].cpu().numpy(), mode, "layer %d" % i)
        plans[i].close()
