"""What the decoder operators' Python entries make of tensors' strides and overlaps."""
import pytest
import torch

import decoder_ref as R
import phi_qlinear as Q

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def batch(dev, lens, Hq=2, H=1, D=64, page=16, dtype=BF16):
    """paged_attention's arguments of a made-up batch, on the device, and its plain form."""
    c = R.make_case(lens, Hq=Hq, H=H, D=D, page=page, dtype=dtype, seed=11)
    want, bound = R.attention(c["q"], c["k"], c["v"], c["ks"], c["vs"], c["table"], c["starts"], c["kv_len"], scale=D ** -0.5)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    args = dict(q=c["q"].to(dev), cache=Q.KvCache(*(c[x].to(dev) for x in ("k", "v", "ks", "vs"))), block_table=c["table"].to(dev),
                q_start=i32(c["starts"]), kv_len=i32(c["kv_len"]), max_q=max(n for n, _ in lens), max_kv=max(kv for _, kv in lens))
    return args, want, bound


def near(got, want, bound):
    return bool(((got.cpu().double() - want).abs() <= bound).all())


def test_table_rows_that_overlap_are_refused(dev):
    """A table of one row for all sequences is no [batch, width] rows in memory."""
    args, want, bound = batch(dev, [(1, 40), (1, 33)])
    table = args.pop("block_table")
    assert near(Q.paged_attention(block_table=table, **args), want, bound)
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device=dev)
    wide[:, :table.shape[1]] = table
    assert near(Q.paged_attention(block_table=wide[:, :table.shape[1]], **args), want, bound)
    with pytest.raises((ValueError, Q.QLinearError), match="block table"):
        Q.paged_attention(block_table=table[:1].expand(2, -1), **args)
    one, want, bound = batch(dev, [(1, 40)])
    table = one.pop("block_table")
    assert near(Q.paged_attention(block_table=torch.as_strided(table, table.shape, (0, 1)), **one), want, bound)
