"""The prompt pass's operators at the edges of what their calls allow."""

import pytest
import torch

from sluice_b200 import _lib, prompt

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


# ------------------------------------------------------------ block planner
@pytest.mark.parametrize("bs", [64, 48, 1])
def test_plan_of_a_context_past_its_complete_table_row(bs):
    """Without a ring, the cached rows behind the table row's last block have
    no slot; those before it, and the requests beside, keep theirs."""
    width = 4
    table = torch.tensor([[5, 9, 2, 7], [1, 0, 3, 4]], **I32)
    context, new = [width * bs + 2 * bs + 3, bs], [1, 2 * bs]
    T, Tk = sum(new), sum(context) + sum(new)
    p = prompt.plan_kv_blocks(torch.tensor(context, **I32), torch.tensor(new, **I32), table,
                              None, None, bs, T, num_kv_tokens=Tk)
    ids = table.tolist()

    def slot(r, q):
        return ids[r][q // bs] * bs + q % bs if q < width * bs else -1

    assert p.status.tolist() == [_lib.KV_PLAN_BAD_INPUT, 0]
    assert p.slots.tolist() == [-1] + [slot(1, q) for q in range(bs, 3 * bs)]
    assert p.positions.tolist() == [context[0]] + list(range(bs, 3 * bs))
    assert p.kv_slots.tolist() == [slot(0, q) for q in range(context[0])] + [-1] + \
        [slot(1, q) for q in range(3 * bs)]
    assert table.tolist() == ids


def test_plan_of_a_context_past_its_row_among_many():
    """The same in several CTAs, several rows a lane."""
    bs, width, B = 16, 3, 700
    context = [width * bs + 100 if r % 3 == 0 else 20 for r in range(B)]
    table = torch.arange(B * width, **I32).view(B, width)
    p = prompt.plan_kv_blocks(torch.tensor(context, **I32), torch.ones(B, **I32), table, None, None,
                              bs, B, num_kv_tokens=sum(context) + B)
    assert p.status[0].item() == _lib.KV_PLAN_BAD_INPUT
    want, want_kv = [], []
    for r, c in enumerate(context):
        rows = [(r * width + q // bs) * bs + q % bs if q < width * bs else -1 for q in range(c + 1)]
        want_kv += rows
        want.append(rows[-1])
    assert p.slots.tolist() == want and p.kv_slots.tolist() == want_kv
