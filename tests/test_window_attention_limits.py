"""artemis_amd.window_attention where its sizes end: an axis next to 2^31 tokens."""
import pytest
import torch

import artemis_amd
import ops_reference as ref

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("axis", [0, 1, 2])
def test_a_shift_past_2_31(axis):
    """Positions in front of the wrap pass 2^31 - 1.  The window that wraps around holds the last position and the first four,
    as on a map of ten."""
    n, small = 2147483645, 10                                # both multiples of 5

    def on(size):
        return tuple(size if i == axis else 1 for i in range(3))

    g = torch.Generator().manual_seed(61)
    values = torch.randn(5, 12, generator=g).bfloat16()      # of the last position, then the first four
    table = torch.randn(9, 1, generator=g)
    qkv = torch.zeros(1, *on(n), 12, dtype=torch.bfloat16, device=DEV)
    flat = qkv.view(n, 12)
    flat[n - 1], flat[:4] = values[0].to(DEV), values[1:].to(DEV)
    labels = torch.zeros(on(n), dtype=torch.int32, device=DEV)
    labels.view(-1)[2] = 1
    shift = on(5)
    shift = tuple(4 if s == 5 else 0 for s in shift)
    out = artemis_amd.window_attention(qkv, table.to(DEV), on(5), 1, labels=labels, shift=shift, outside=-1.5).view(n, 4)
    got = torch.cat([out[n - 1:], out[:4]])
    assert float(out[4:1000].abs().max()) == 0 and float(out[n - 1000:n - 1].abs().max()) == 0
    del qkv, flat, labels, out
    torch.cuda.empty_cache()
    few = torch.zeros(small, 12, dtype=torch.bfloat16)
    few[small - 1], few[:4] = values[0], values[1:]
    lab = torch.zeros(small, dtype=torch.int32)
    lab[2] = 1
    want, bound = ref.window_attention(few.view(1, *on(small), 12), table, on(5), 1, shift=shift, labels=lab.view(on(small)),
                                       outside=-1.5)["out"]
    order = [small - 1, 0, 1, 2, 3]
    ref.assert_within(got, want.view(small, 4)[order], bound.view(small, 4)[order], "out")
