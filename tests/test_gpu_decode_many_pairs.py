"""Batched decode of contiguous caches with more (sequence, KV head) pairs than
workgroups are resident at once: every pair's output is written."""
import numpy as np
import pytest

from oracle import oracle as orc

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("batch,hk,group", [(64, 16, 1), (50, 32, 2), (64, 40, 1)])
def test_every_pair_is_attended(batch, hk, group):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import turboquant_amd as tq
    d, bits, cap, rng = 64, 3, 1100, np.random.default_rng(batch)
    lens = rng.integers(1, cap + 1, size=batch)
    lens[0], lens[-1] = cap, 900
    g = torch.Generator(device="cuda").manual_seed(1)
    recs = []
    for _ in range(2):
        p, s = tq.pqo_quantize(torch.randn(batch * hk * cap, d, generator=g, device="cuda"), bits)
        recs += [p.view(batch, hk, cap, -1), s.view(batch, hk, cap, -1)]
    q = torch.randn(batch, hk * group, d, generator=g, device="cuda")
    ws = tq.AttentionWorkspace(batch, hk * group, hk, d, cap)
    out = torch.full((batch, hk * group, d), float("nan"), device="cuda")
    tq.pqo_decode_attention(q, *recs, torch.from_numpy(lens.astype(np.int32)).cuda(), hk, bits, cap, cap, hk * cap,
                            d ** -0.5, ws, out=out)
    assert not out.isnan().any(), f"{int(out.isnan().any(-1).sum())} of {batch * hk * group} rows not written"
    for b in (0, batch // 2, batch - 1):
        n = int(lens[b])
        k, v = (orc.pqo_dequantize(bits, recs[i][b, :, :n].cpu().numpy().reshape(hk * n, -1),
                                   recs[i + 1][b, :, :n].cpu().numpy().view(np.uint16).reshape(hk * n, -1), d)
                .reshape(hk, n, d) for i in (0, 2))
        ref = orc.attention_dense(q[b].cpu().numpy(), k, v, d ** -0.5)
        assert np.abs(out[b].cpu().numpy() - ref).max() <= 1e-3
