"""Workspaces of cross attention: every shape whose keys the library splits gets one."""
from __future__ import annotations

import pytest
import torch

from test_gpu_cross import F, U, Plain

pytestmark = pytest.mark.gpu


# batch x heads of 514 to 591 tiles of up to 256 rows, just under four per SM, with keys long enough to be split
@pytest.mark.parametrize("size", [(11, 250, 32768, 48, 1, 64), (43, 256, 16384, 12, 1, 128), (66, 256, 32768, 8, 1, 64),
                                  (67, 240, 65536, 8, 1, 128), (37, 190, 40000, 15, 1, 64)])
def test_split_keys_of_many_tiles(size):
    import htrc_b200
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    b, n, m, h, hk, d = size
    gen = torch.Generator(device="cuda").manual_seed(n)
    q = torch.randn((b, h, n, d), generator=gen, device="cuda").bfloat16()
    k, v = (torch.randn((b, hk, m, d), generator=gen, device="cuda").bfloat16() for _ in range(2))
    out, lse = htrc_b200.cross_attention(q, k, v, heads_first=True, return_lse=True)
    htrc_b200.cross_status()
    u = U[q.dtype]
    for i, j in ((0, 0), (b // 2, h - 1), (b - 1, h // 2)):
        ref = Plain(q[i:i + 1, j:j + 1], k[i:i + 1], v[i:i + 1])
        assert ((out[i, j] - ref.out[0, 0]).abs() <= u * ref.out[0, 0].abs() + (u + F) * ref.out_bound[0, 0]).all()
        assert ((lse[i, j] - ref.lse[0, 0]).abs() <= 2.0 ** -18 * (1 + ref.s[0, 0].abs().amax(-1))).all()
