"""append_paged against the float64 oracle: every other row of the pages stays as it was."""

import numpy as np
import pytest
import torch

from cab_attention.cache import append_paged
from cab_attention.kernels import Rotary
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rand(shape, dt, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(DT[dt])


def np64(t):
    return t.detach().double().cpu().numpy()


CASES = [  # B, H, H_kv, n, D, S, lengths, counts
    (1, 4, 4, 1, 64, 16, [0], None),                       # the first row of all
    (3, 8, 2, 1, 128, 16, [15, 16, 31], None),             # last and first places of a page
    (2, 3, 1, 5, 64, 4, [2, 7], [5, 0]),                   # over three pages; none
    (3, 4, 2, 40, 128, 24, [0, 23, 50], [40, 17, 99]),     # counts past n
    (4, 2, 2, 3, 64, 1, [-1, 5, 6, 2 ** 31 - 2], None),    # a page a row; negative and past the table
    (2, 2, 1, 6, 50, 5, [1, 17], [3, -4]),                 # rows off 16-byte boundaries
    (1, 28, 4, 1100, 128, 64, [37], None),                 # four tokens a workgroup
    (2, 0, 1, 7, 511, 3, [4, 0], None),                    # no queries; the widest, value by value
]


def setup(case, dt, cuda, seed=0):
    B, H, Hkv, n, D, S, lengths, counts = case
    rng = np.random.default_rng(seed)
    columns = max(2, -(-(max(min(x, 2000) for x in lengths) + n) // S) - (S == 1))
    pages = B * columns + 2
    table = rng.permutation(pages)[:B * columns].reshape(B, columns)
    pools = [rand((pages, Hkv, S, D), dt, 1), rand((pages, Hkv, S, D), dt, 2)]
    k, v = rand((B, n, Hkv, D), dt, 3).transpose(1, 2), rand((B, Hkv, n, D), dt, 4)
    q = rand((B, n, H, D), dt, 5).transpose(1, 2) if H else None
    dev = lambda t: None if t is None else t.to(cuda)
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=cuda)
    return (k, v, q, pools, table), dict(k=dev(k), v=dev(v), k_pages=dev(pools[0]), v_pages=dev(pools[1]),
                                         page_table=i32(table), lengths=i32(lengths), counts=i32(counts))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rows_as_they_are(cuda, case, dt):
    (k, v, q, pools, table), a = setup(case, dt, cuda)
    before = a["k_pages"]._version
    assert append_paged(**a) is None
    for new, pool, got in ((k, pools[0], a["k_pages"]), (v, pools[1], a["v_pages"])):
        want = P.append(np64(pool), np64(new), table, case[6], case[7])
        np.testing.assert_array_equal(np64(got), want)
    assert a["k_pages"]._version > before


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", CASES, ids=str)
def test_rotated(cuda, case, dt, interleaved):
    """K and q as Rotary turns them at the rows' own numbers, bit for bit; V as it is."""
    (k, v, q, pools, table), a = setup(case, dt, cuda)
    B, H, Hkv, n, D, S, lengths, counts = case
    rot = Rotary(D, rotary_dim=D // 4 * 2, interleaved=interleaved,
                 scaling=dict(type="yarn", factor=2.0, original_length=512)).to(cuda)
    at = torch.tensor(lengths)[:, None] + torch.arange(n)
    # (int64: the sum passes 32 bits only in rows that go nowhere)
    at = at.clamp(max=2 ** 31 - 1).to(cuda)
    got_q = append_paged(**a, rotary=rot, q=None if q is None else q.to(cuda))
    turned = rot(k.to(cuda), positions=at)
    np.testing.assert_array_equal(np64(a["k_pages"]), P.append(np64(pools[0]), np64(turned), table, lengths, counts))
    np.testing.assert_array_equal(np64(a["v_pages"]), P.append(np64(pools[1]), np64(v), table, lengths, counts))
    if q is not None:
        want = rot(q.to(cuda), positions=at)
        fits = [b for b in range(B) if lengths[b] + n < 2 ** 31]
        assert torch.equal(got_q[fits], want[fits]) and got_q.stride() == want.stride()


def test_given_positions(cuda):
    """A cache that has dropped rows: positions run ahead of the rows; one list, or one a sequence."""
    case = (2, 4, 2, 3, 64, 16, [5, 14], None)
    (k, v, q, pools, table), a = setup(case, "bf16", cuda)
    rot = Rotary(64).to(cuda)
    for at in ([[1000, 1001, 1002], [70, 71, 72]], [9, 8, 7]):
        a["k_pages"].copy_(pools[0])
        at = torch.tensor(at, device=cuda)
        got_q = append_paged(**a, rotary=rot, q=q.to(cuda), positions=at)
        assert torch.equal(got_q, rot(q.to(cuda), positions=at))
        np.testing.assert_array_equal(np64(a["k_pages"]),
                                      P.append(np64(pools[0]), np64(rot(k.to(cuda), positions=at)), table, [5, 14]))


def test_pages_that_are_not_there(cuda):
    case = (3, 0, 2, 8, 64, 4, [1, 2, 3], None)
    (k, v, _, pools, table), a = setup(case, "fp16", cuda)
    table = table.copy()
    table[0, 1], table[1, 0], table[2, 2], table[2, 1] = -1, pools[0].shape[0], 2 ** 31 - 1, -2 ** 31
    a["page_table"] = torch.tensor(table, device=cuda)  # int64, converted
    append_paged(**a)
    np.testing.assert_array_equal(np64(a["k_pages"]), P.append(np64(pools[0]), np64(k), table, [1, 2, 3]))
    np.testing.assert_array_equal(np64(a["v_pages"]), P.append(np64(pools[1]), np64(v), table, [1, 2, 3]))


def test_layouts(cuda):
    """Pools laid out [P, S, H, D], K and V side by side, a table that is a part of a larger one."""
    case = (3, 4, 2, 5, 64, 8, [3, 9, 0], None)
    (k, v, q, pools, table), a = setup(case, "bf16", cuda)
    P_, Hkv, S, D = pools[0].shape
    both = torch.zeros((P_, S, Hkv, 2, D), dtype=torch.bfloat16, device=cuda)
    kp, vp = both[:, :, :, 0].transpose(1, 2), both[:, :, :, 1].transpose(1, 2)
    kp.copy_(pools[0])
    vp.copy_(pools[1])
    big = torch.full((9, table.shape[1] + 3), -1, dtype=torch.int32, device=cuda)
    big[2:5, 1:1 + table.shape[1]] = a["page_table"]
    a.update(k_pages=kp, v_pages=vp, page_table=big[2:5, 1:1 + table.shape[1]])
    qkv = torch.cat([x.to(cuda).transpose(1, 2) for x in (q, k, v)], 2)  # one projection's result
    a.update(k=qkv[:, :, 4:6].transpose(1, 2), v=qkv[:, :, 6:].transpose(1, 2))
    rot = Rotary(64).to(cuda)
    got_q = append_paged(**a, rotary=rot, q=qkv[:, :, :4].transpose(1, 2))
    at = (torch.tensor(case[6])[:, None] + torch.arange(5)).to(cuda)
    assert torch.equal(got_q, rot(q.to(cuda), positions=at))
    np.testing.assert_array_equal(np64(kp), P.append(np64(pools[0]), np64(rot(k.to(cuda), positions=at)), table, case[6]))
    np.testing.assert_array_equal(np64(vp), P.append(np64(pools[1]), np64(v), table, case[6]))


def test_nan_rows_are_copied_bit_for_bit(cuda):
    (k, v, _, pools, table), a = setup((1, 0, 1, 2, 64, 16, [3], None), "bf16", cuda)
    bits = torch.full((1, 1, 2, 64), 0x7fab, dtype=torch.int16, device=cuda)
    a["v"] = bits.view(torch.bfloat16)
    append_paged(**a, rotary=Rotary(64).to(cuda))
    got = a["v_pages"].view(torch.int16)[int(table[0, 0]), :, 3:5]
    assert (got == 0x7fab).all()


def test_empty_calls(cuda):
    (k, v, q, pools, table), a = setup((2, 4, 2, 3, 64, 16, [0, 5], None), "bf16", cuda)
    rot = Rotary(64).to(cuda)
    none = dict(a, k=a["k"][:, :, :0], v=a["v"][:, :, :0])
    assert append_paged(**none, rotary=rot, q=q.to(cuda)[:, :, :0]).shape == (2, 4, 0, 64)
    no_columns = dict(a, page_table=a["page_table"][:, :0])
    at = (torch.tensor([0, 5])[:, None] + torch.arange(3)).to(cuda)
    assert torch.equal(append_paged(**no_columns, rotary=rot, q=q.to(cuda)), rot(q.to(cuda), positions=at))
    no_pages = dict(a, k_pages=a["k_pages"][:0], v_pages=a["v_pages"][:0])
    append_paged(**no_pages)
    assert torch.equal(a["k_pages"].cpu(), pools[0])


def test_refusals_on_the_device(cuda):
    (k, v, q, pools, table), a = setup((2, 4, 2, 3, 64, 16, [0, 5], None), "bf16", cuda)
    rot = Rotary(64).to(cuda)
    for change, error, match in (
            (dict(v_pages=a["k_pages"]), ValueError, "share memory"),
            (dict(k=a["k_pages"][:2, :, :3]), ValueError, "share memory"),
            (dict(k_pages=a["k_pages"][..., :1].expand(-1, -1, -1, 64)), ValueError, "stride"),
            (dict(k_pages=a["k_pages"][:, :, :1].expand(-1, -1, 16, -1)), ValueError, "overlap"),
            (dict(page_table=a["page_table"][0]), ValueError, "page_table"),
            (dict(page_table=a["page_table"].float()), TypeError, "page_table"),
            (dict(lengths=a["lengths"][:1]), ValueError, "lengths"),
            (dict(counts=a["lengths"].cpu()), RuntimeError, "GPU"),
            (dict(q=q.to(cuda)), ValueError, "rotary"),
            (dict(rotary=Rotary(128).to(cuda)), ValueError, "heads"),
            (dict(rotary=Rotary(64)), RuntimeError, "GPU"),
            (dict(rotary=rot, q=q.to(cuda)[:, :, :2]), ValueError, "q must be"),
            (dict(rotary=rot, q=q.to(cuda).half()), TypeError, "dtypes"),
            (dict(k=a["k"].clone().requires_grad_()), RuntimeError, "gradient")):
        with pytest.raises(error, match=match):
            append_paged(**{**a, **change})
    assert torch.equal(a["k_pages"].cpu(), pools[0]) and torch.equal(a["v_pages"].cpu(), pools[1])
    with torch.inference_mode():
        closed = a["k_pages"].clone()
    with pytest.raises(RuntimeError, match="inference"):
        append_paged(**dict(a, k_pages=closed))
