"""Attention in fp16 where one key takes nearly all the weight and the others' values make the result: weights a few
millionths of the largest have to keep their bits.

The bound is that of the definition's weights p and values v: u |o| + (2^-11 + 2 e) sum p|v| for one rounding of the
output, one of each weight to fp16, and e for what 32 bits and the hardware's exponential move a weight by; and, since
fp16 has steps of 2^-24 at the least, 2^-32 max p sum |v|: half such a step of weights that are taken 2^7 times higher
than the largest. The output's own least step adds 2^-25."""

from __future__ import annotations

import math

import pytest
import torch
from paged_oracle import HALF_STEP, Problem, sees

from ako_b200 import paged_attention_cuda_sm100

pytestmark = pytest.mark.gpu

F16 = torch.float16


@pytest.mark.parametrize("bits", [16.3, 20.6, 23.4])
@pytest.mark.parametrize("quantised", [False, True], ids=["same", "e4m3"])
@pytest.mark.parametrize("new", [1, 3, 8, 100], ids=["8rows", "16rows", "32rows", "many"])
def test_weights_far_below_the_largest(cuda_device, bits, quantised, new) -> None:
    """Values of some hundreds; the first key's are 2^-9 of them or less. In e4m3 all scales are the same, as a caller
    has them who scales a whole cache by one number."""
    kv, dim = 900, 128
    p = Problem(F16, quantised, 8, 2, dim, 16, [(new, kv)], True, 61, cuda_device)
    p.q[..., 0] = 1.0
    pull = bits * math.log(2.0) * math.sqrt(dim)
    g = torch.Generator().manual_seed(62)
    v = torch.randint(128, 449, (kv, 2, dim), generator=g).double()
    if quantised:
        v = (v / 32).round() * 32  # on e4m3's grid up to 448
    v[0] = 0.25
    for j in range(kv):
        at = int(p.table[0, j // 16]), slice(None), j % 16
        if quantised:
            for name in ("k", "v"):
                p.caches[name + "_scale"][at] = 1.0 if name == "v" else pull / 448 if j == 0 else 2.0**-9
            p.caches["v"][at] = v[j].to(device=cuda_device, dtype=torch.float32).to(torch.float8_e4m3fn)
            k = p.caches["k"][at].float().cpu()
            k[:, 0] = 0.0
            if j == 0:
                k[:] = 0.0
                k[:, 0] = 448.0
            p.caches["k"][at] = k.to(cuda_device).to(torch.float8_e4m3fn)
            p.k[0][j] = k.double() * p.caches["k_scale"][at].double().cpu()[:, None]
        else:
            p.k[0][j, :, 0] = 0.0
            if j == 0:
                p.k[0][j] = 0.0
                p.k[0][j, :, 0] = float(torch.tensor(pull).to(F16))
            p.caches["k"][at] = p.k[0][j].to(F16).to(cuda_device)
            p.caches["v"][at] = v[j].to(F16).to(cuda_device)
    got = paged_attention_cuda_sm100(p.q.to(cuda_device), p.kv(), p.batch(new)).double().cpu()
    ok = sees(new, kv, 0, 0)
    for h in range(8):
        k, values = p.k[0][:, h // 4], v[:, h // 4]
        q = p.q[:, h].double()
        s = (q @ k.T * dim**-0.5).masked_fill(~ok, -math.inf)
        w = torch.softmax(s, -1)
        size = (q.abs() @ k.abs().T * dim**-0.5).masked_fill(~ok, 0.0)
        e = ((dim + 4) * 2.0**-24 * size + 4 * 2.0**-24 * s.masked_fill(~ok, 0.0).abs()).amax(-1, keepdim=True)
        e = e + 2.0**-20 + kv * 2.0**-23
        want = w @ values
        bound = (HALF_STEP[F16] * want.abs() + (2.0**-11 + 2 * e) * want
                 + 2.0**-32 * w.amax(-1, keepdim=True) * (ok.double() @ values) + 2.0**-25)
        others = w[:, 1:] @ values[1:]
        assert float((others / bound).median()) > 4  # the bound sees whether the others' weights are there
        over = float(((got[:, h] - want).abs() / bound).max())
        assert over <= 1.0, f"head {h}: {over:.2f} of the bound"
