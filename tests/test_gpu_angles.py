"""How exact the angles of the rotation are."""
import numpy as np
import pytest
import torch

from attention_plain import EPS, to64
from diskmule_b200 import CudaContext, _native as N
from diskmule_b200.attention import Rope, rotate
from paged import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("position", [1, 1000003, 2 ** 31 - 1])
@pytest.mark.parametrize("turns", [0.0, 0.5, 30.5])
def test_angles_near_whole_and_half_turns(position, turns):
    """Where the sine is near zero its 16 bits show an angle that is off by 2^-25 of a turn (2 pi 2^-25
    in the sine), beside the result's own rounding; the sine has two units of 2^-24 of itself. The
    angle of the 64-bit frequency is taken in whole numbers: it is `turns` and a little more."""
    ctx = CudaContext(0)
    r = np.random.RandomState(position % 1000)
    little = np.ldexp(r.uniform(1, 2, 128), r.randint(-22, -9, 128)) * r.choice([-1, 1], 128)
    f = 2 * np.pi * (turns + little) / position
    # the angle that these 64 bits stand for, modulo one turn, with pi to 2^-100
    pi = 0x3243F6A8885A308D313198A2E  # times 2^-96
    exact = []
    for x in f:
        m, e = np.frexp(x)
        whole = (int(m * 2 ** 53) * position << 200) * 2 ** 96 // (2 * pi)  # turns times 2^(200 + 53 - e)
        bits = 200 + 53 - int(e)
        part = whole % (1 << bits)
        if 2 * part > 1 << bits:
            part -= 1 << bits
        exact.append(part / 2 ** bits)
    exact = np.array(exact)
    rope = Rope(ctx, 256, frequencies=f)
    q = torch.zeros(1, 1, 256, dtype=torch.bfloat16, device="cuda")
    q[..., :128] = 1
    out, at = torch.empty_like(q), ints([position])
    rotate(ctx, rope, type=N.BF16, head_dim=256, tokens=1, heads=1, q=q.data_ptr(), q_out=out.data_ptr(),
           positions=at.data_ptr())
    torch.cuda.synchronize()
    got, want = to64(out)[0, 0, 128:], np.sin(2 * np.pi * exact)
    off = 2 * np.pi * 2.0 ** -25
    assert np.all(np.abs(got - want) <= off + (EPS[torch.bfloat16] + 2.0 ** -22) * (np.abs(want) + off))
    rope.close()
    ctx.close()
