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


@pytest.mark.parametrize("lens", [[(1, 50), (1, 33)], [(140, 200), (3, 90)]])
@pytest.mark.parametrize("within", ["tokens", "heads"])
def test_attention_output_beside_its_queries(dev, lens, within):
    """q and out as columns of one tensor that share no element."""
    args, want, bound = batch(dev, lens, Hq=4)
    q = args.pop("q")
    T, Hq, D = q.shape
    both = torch.full((T, 2 * Hq, D) if within == "tokens" else (T, Hq, 2 * D), 9.0, dtype=BF16, device=dev)
    left, right = both.split(Hq, dim=1) if within == "tokens" else both.split(D, dim=2)
    left.copy_(q)
    # The plain bound is for exact keys: chunks round them to 11 bits, which 2^-9 of the weights' sum covers here.
    got = Q.paged_attention(left, out=right, **args)
    assert got.data_ptr() == right.data_ptr() and torch.equal(left, q)
    assert torch.equal(right, Q.paged_attention(q, **args)) and bool(((got.cpu().double() - want).abs() <= bound + 2.0 ** -6).all())


def test_norm_on_columns_of_one_tensor(dev):
    """x, its residual stream (updated in place) and the normalised row side by side."""
    rows, K = 37, 512
    wide = torch.randn((rows, 3 * K), generator=torch.Generator().manual_seed(2)).to(dev)
    x, h, y = wide.split(K, dim=1)
    x0, h0 = x.clone(), h.clone()
    new, y0 = torch.empty_like(h0), torch.empty_like(h0)
    w = torch.linspace(0.5, 1.5, K, device=dev)
    q0, s0 = Q.rms_norm_quant(x0, w, 1e-6, residual=h0, residual_out=new, y=y0)
    q, s = Q.rms_norm_quant(x, w, 1e-6, residual=h, residual_out=h, y=y)
    assert torch.equal(q, q0) and torch.equal(s, s0) and torch.equal(x, x0) and torch.equal(h, new) and torch.equal(y, y0)


# ------------------------------------------------------------------ rows without a norm
@pytest.mark.parametrize("K,rotate", [(512, True), (4096, True), (1000, False), (20480, False)])
@pytest.mark.parametrize("ydtype", [BF16, F32])
def test_norm_rows_that_are_not_finite(dev, K, rotate, ydtype):
    """Where a row's scale is NaN its normalised row is too, in every place: an
    infinity or a NaN in it, or squares whose sum passes 32 bits."""
    x = torch.randn((6, K), generator=torch.Generator().manual_seed(K))
    x[1, 3], x[2, K - 1], x[4, K // 2] = torch.inf, torch.nan, -torch.inf
    x[3] *= 1e20
    y = torch.zeros((6, K), dtype=ydtype, device=dev)
    shift = torch.ones(K, device=dev)
    q, s = Q.rms_norm_quant(x.to(dev), None, 1e-6, shift=shift, rotate=rotate, y=y)
    bad = torch.tensor([False, True, True, True, True, False])
    assert torch.equal(s.cpu().isnan(), bad) and not q.cpu()[bad].any()
    assert torch.equal(y.cpu().isnan(), bad[:, None].expand(6, K))
