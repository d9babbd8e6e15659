"""4-bit attention of few heads in calls that take several launches, cut inside sequences too, against 64 bits."""
import pytest
import torch

from llmdivedeep_b200 import ops
from oracle import latent4_oracle as L
from tests.test_gpu_latent4 import MOST, REL, rope_bytes

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,tokens,H,K", [(160001, 160001, 2, 3), (140002, 70001, 1, 5), (75799, 7, 1, 3), (80000, 80000, 17, 70)])
@pytest.mark.parametrize("room", [True, False])
def test_calls_of_several_launches(T, tokens, H, K, room):
    g = torch.Generator(device="cuda").manual_seed(T)
    B, P = -(-T // tokens), 3
    kv = torch.randn(40 * 64, 576, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    rec = torch.from_numpy(L.records(kv.double().numpy(), rope_bytes(kv))).cuda()
    table = torch.randint(0, 40, (B, P), device="cuda", generator=g, dtype=torch.int32)
    q = torch.randn(T, H, 576, device="cuda", generator=g, dtype=torch.bfloat16)
    # distinct positions; a row in seven selects nothing, others have holes
    first = torch.randint(0, P * 64, (T, 1), device="cuda", generator=g)
    idx = ((first + torch.arange(K, device="cuda") * 11) % (P * 64)).int()
    idx[torch.rand(T, K, device="cuda", generator=g) < 0.2] = -1
    idx[3::7] = -1
    ws = None if room else torch.empty(0, dtype=torch.uint8, device="cuda")
    out = torch.full((T, H, 512), 9.0, dtype=torch.bfloat16, device="cuda")
    ops.sparse_mla_decode_paged(q, rec, table, idx, 192 ** -0.5, out=out, workspace=ws, tokens_per_seq=tokens)
    ops.check_status("cuda")
    values = torch.from_numpy(L.decode(rec.cpu().numpy())).cuda()
    for r0 in range(0, T, 4000):
        rows = torch.arange(r0, min(T, r0 + 4000), device="cuda")
        pos = idx[rows].long()
        at = pos.clamp_min(0)
        x = values[table[rows // tokens].long().gather(1, at // 64) * 64 + at % 64]
        s = (torch.einsum("thd,tkd->thk", q[rows].double(), x) * 192 ** -0.5).masked_fill((pos < 0)[:, None], float("-inf"))
        want = torch.einsum("thk,tkd->thd", torch.softmax(s, -1).nan_to_num(0.0), x[..., :512])
        got = out[rows].double()
        err, size = (got - want).norm(dim=-1), want.norm(dim=-1)
        assert bool((err <= REL * size).all()), (r0, float((err / size.clamp_min(1e-30)).max()))
        assert bool(((got - want).abs().amax(-1) <= MOST * want.abs().amax(-1)).all())
