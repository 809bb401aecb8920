"""adjust_logits against the float64 oracle: histories, prompts, penalties, biases, masks, trees."""

import numpy as np
import pytest
import torch

from cab_attention.kernels import adjust_logits
from oracle import paged_oracle as P

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def np64(t):
    return t.detach().double().cpu().numpy()


def pack(allowed, cuda):
    """Truth values [.., V] as words of 32 bits."""
    V = allowed.shape[-1]
    bits = np.zeros((*allowed.shape[:-1], -(-V // 32) * 32), dtype=np.uint8)
    bits[..., :V] = allowed
    words = np.packbits(bits, axis=-1, bitorder="little").view("<i4")
    return torch.tensor(words.astype(np.int32), device=cuda)


def setup(B, T, V, L, dt, seed=0, biases=0, masked=False, tree=False, per_sequence=True):
    rng = np.random.default_rng(seed)
    a = dict(logits=torch.tensor(3 * rng.normal(size=(B, T, V))).to(DT[dt]))
    if L:
        words = (rng.random((B, L)) ** 3 * V).astype(int)
        words[rng.random((B, L)) < 0.05] = V + 3      # outside the vocabulary
        words[rng.random((B, L)) < 0.05] = -1
        a["history"] = words
        a["lengths"] = rng.integers(0, L + 1, B)
        a["prompts"] = rng.integers(0, L + 1, B)
    for name, x in (("repetition", 1 + 0.5 * rng.random(B)), ("presence", rng.normal(size=B)),
                    ("frequency", 0.3 * rng.random(B))):
        a[name] = x.astype(np.float32) if per_sequence else float(np.float32(x[0]))
    if biases:
        a["bias_tokens"] = rng.integers(-2, V + 2, (B, biases))
        a["bias_tokens"][:, -1] = a["bias_tokens"][:, 0]  # listed twice
        a["bias"] = (4 * rng.normal(size=(B, biases))).astype(np.float32)
    if masked:
        a["allowed"] = rng.random((B, T, V)) < 0.3
    if tree:
        a["drafts"] = (rng.random((B, T)) ** 3 * (V + 2)).astype(int)
        a["drafts"][:, -1] = a["drafts"][:, 0]
        a["parents"] = np.array([[-1 if i == 0 else int(i * rng.random()) for i in range(T)] for _ in range(B)])
        if T > 3:
            a["parents"][0, T - 2] = -2
            a["parents"][0, T - 1] = T - 2
    return a


def call(a, cuda, **more):
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device=cuda)
    f32 = lambda x: torch.tensor(x, device=cuda) if isinstance(x, np.ndarray) else x
    kw = dict(history=i32(a.get("history")), lengths=i32(a.get("lengths")), prompt_lengths=i32(a.get("prompts")),
              repetition=f32(a["repetition"]), presence=f32(a["presence"]), frequency=f32(a["frequency"]),
              bias_tokens=i32(a.get("bias_tokens")), bias=None if "bias" not in a else f32(a["bias"]),
              allowed=None if "allowed" not in a else pack(a["allowed"], cuda),
              drafts=None if "drafts" not in a else torch.tensor(a["drafts"], device=cuda),
              parents=i32(a.get("parents")))
    return adjust_logits(a["logits"].to(cuda), **{**kw, **more})


def check(a, got, dt):
    want = P.adjust(np64(a["logits"]), **{k: v for k, v in a.items() if k != "logits"})
    low = np.isneginf(want)
    got = np64(got)
    assert np.array_equal(np.isneginf(got), low)
    # fp32: a quotient or product, the penalties' product and two sums, the bias's: five
    # roundings of values below `big`; then half a step of the type.
    n = a["history"].shape[1] if "history" in a else 0
    big = np.abs(np64(a["logits"])).max() * 1.5 + 5 + 0.3 * (n + 256) + 20
    np.testing.assert_allclose(got[~low], want[~low], rtol=torch.finfo(DT[dt]).eps / 2 * (1 + 1e-6),
                               atol=5 * 2.0 ** -24 * big)
    return low


CASES = [  # B, T, V, L, biases, masked, tree
    (1, 1, 1, 1, 1, False, False),           # one token
    (1, 1, 7, 5, 2, True, False),
    (2, 1, 32, 0, 0, True, False),           # a mask alone
    (3, 1, 1000, 100, 0, False, False),
    (2, 1, 1024, 33, 5, False, False),       # a stretch, exactly
    (2, 1, 1025, 33, 5, True, False),        # and one more
    (1, 1, 32000, 600, 10, False, False),
    (2, 1, 50001, 5003, 0, True, False),     # odd rows
    (4, 3, 4097, 50, 300, True, True),
    (1, 26, 20001, 2000, 7, True, True),
    (40, 2, 33000, 64, 0, False, True),      # long stretches
    (2, 256, 301, 20, 3, True, True),        # the most nodes
    (3, 5, 2000, 0, 0, False, True),         # drafts alone
    (2, 4, 999, 40, 2, True, False),         # several rows without a tree
]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", CASES, ids=str)
def test_against_the_oracle(cuda, case, dt):
    B, T, V, L, biases, masked, tree = case
    a = setup(B, T, V, L, dt, biases=biases, masked=masked, tree=tree)
    check(a, call(a, cuda), dt)


def test_one_value_for_all_and_defaults(cuda):
    a = setup(3, 1, 500, 40, "fp32", per_sequence=False)
    check(a, call(a, cuda), "fp32")
    x = a["logits"].to(cuda)
    assert torch.equal(adjust_logits(x), x)
    h = torch.tensor(a["history"], device=cuda)  # int64, whole
    assert torch.equal(adjust_logits(x, h), x)
    assert torch.equal(adjust_logits(x, h, presence=0.5), adjust_logits(x, h.int(), presence=0.5))
    check(dict(a, lengths=None, prompts=None), adjust_logits(
        x, h, repetition=a["repetition"], presence=a["presence"], frequency=a["frequency"]), "fp32")


def test_mask_for_all_nodes_and_one_tree(cuda):
    a = setup(3, 6, 700, 20, "fp16", biases=2, masked=True, tree=True)
    a["allowed"][:] = a["allowed"][:, :1]
    a["parents"][:] = a["parents"][:1]
    one = call(a, cuda, allowed=pack(a["allowed"][:, 0], cuda),
               parents=torch.tensor(a["parents"][0], device=cuda), drafts=torch.tensor(a["drafts"], device=cuda).int())
    check(a, one, "fp16")
    assert torch.equal(one, call(a, cuda))


@pytest.mark.parametrize("dt", list(DT))
def test_untouched_values_keep_their_bits(cuda, dt):
    """NaN and infinities pass; a masked one is -inf; a row without any allowed token is all -inf."""
    a = setup(2, 2, 999, 30, dt, masked=True)
    x = a["logits"]
    x[0, 0, :5] = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0, 0.0])
    x[0, 1, 990:] = float("nan")
    a["allowed"][0, 0, :5] = True
    a["allowed"][1, 1] = False
    a["history"][:] = 7
    got = call(a, cuda).cpu()
    bits = torch.int32 if dt == "fp32" else torch.int16
    keep = torch.tensor(a["allowed"])
    keep[:, :, 7] = False
    assert torch.equal(got.view(bits)[keep], x.view(bits)[keep])
    gone = ~torch.tensor(a["allowed"])
    assert torch.isneginf(got[gone]).all() and torch.isneginf(got[1, 1]).all()


def test_infinite_logits_and_overflow(cuda):
    x = torch.tensor([[[float("inf"), -float("inf"), 60000.0, -60000.0, 2.0]]], dtype=torch.float16, device=cuda)
    h = torch.arange(5, device=cuda)[None].int()
    got = adjust_logits(x, h, repetition=2.0, presence=1.0)
    assert got[0, 0].tolist() == [float("inf"), -float("inf"), 30000.0, -float("inf"), 0.0]


def test_layouts_and_out(cuda):
    """Rows of a larger tensor at any alignment, out in place or elsewhere, a history that is a part of
    a larger one, off 16-byte boundaries."""
    a = setup(2, 3, 1501, 70, "bf16", biases=3, masked=True, tree=True)
    want = call(a, cuda)
    x = a["logits"].to(cuda)
    for lead in (0, 1, 3, 8):
        room = torch.zeros((2, 5, 1501 + 11), dtype=torch.bfloat16, device=cuda)
        view = room[:, 1:4, lead:lead + 1501]
        view.copy_(x)
        assert torch.equal(adjust_like(a, cuda, view), want)
        out = torch.full_like(room, 9.0)
        to = out[:, 2:, lead + 1:lead + 1502]
        assert adjust_like(a, cuda, view, out=to) is to and torch.equal(to, want)
        to.fill_(9.0)
        assert (out == 9.0).all()
        adjust_like(a, cuda, view, out=view)
        assert torch.equal(view, want)
        room[:, 1:4, lead:lead + 1501] = 0
        assert not room.any()
    wide = torch.zeros((2, 79), dtype=torch.int32, device=cuda)
    wide[:, 5:75] = torch.tensor(a["history"], device=cuda)
    assert torch.equal(call(a, cuda, history=wide[:, 5:75]), want)
    flipped = torch.zeros((2, 3, 3002), dtype=torch.bfloat16, device=cuda)[..., ::2]
    flipped.copy_(x)
    assert torch.equal(adjust_like(a, cuda, flipped), want)


def adjust_like(a, cuda, logits, **more):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    return adjust_logits(logits, i32(a["history"]), i32(a["lengths"]), i32(a["prompts"]),
                         *(torch.tensor(a[k], device=cuda) for k in ("repetition", "presence", "frequency")),
                         i32(a["bias_tokens"]), torch.tensor(a["bias"], device=cuda), pack(a["allowed"], cuda),
                         i32(a["drafts"]), i32(a["parents"]), **more)


def test_one_token_a_thousand_times(cuda):
    """Counts from many lanes at once, and a prompt that holds the token too."""
    x = torch.zeros((1, 1, 40), device=cuda)
    h = torch.full((1, 5000), 17, dtype=torch.int32, device=cuda)
    got = adjust_logits(x, h, prompt_lengths=torch.tensor([1000], device=cuda), frequency=0.25, presence=1.0)
    assert float(got[0, 0, 17]) == -1001.0 and not got[0, 0, :17].any() and not got[0, 0, 18:].any()


def test_one_token_in_a_vocabulary(cuda):
    x = torch.ones((2, 1, 9), device=cuda)[:, :, ::5][:, :, :1]
    out = torch.zeros((2, 1, 9), device=cuda)[:, :, ::5][:, :, 1:]
    h = torch.zeros((2, 3), dtype=torch.int32, device=cuda)
    assert adjust_logits(x, h, frequency=2.0, out=out) is out and (out == -5.0).all()
    assert (adjust_logits(x, h, frequency=2.0) == -5.0).all()


def test_empty_calls(cuda):
    for shape in ((0, 1, 10), (2, 0, 10), (2, 1, 0)):
        assert adjust_logits(torch.empty(shape, device=cuda)).shape == shape
    x = torch.ones((2, 1, 10), device=cuda)
    none = torch.zeros((2, 0), dtype=torch.int32, device=cuda)
    assert torch.equal(adjust_logits(x, none, presence=1.0, bias_tokens=none, bias=none.float()), x)


def test_refusals_on_the_device(cuda):
    x = torch.zeros((2, 3, 100), device=cuda)
    h = torch.zeros((2, 5), dtype=torch.int32, device=cuda)
    words = torch.zeros((2, 4), dtype=torch.int32, device=cuda)
    for kw, error, match in (
            (dict(history=h[:1]), ValueError, "history"), (dict(history=h.float()), TypeError, "history"),
            (dict(lengths=h[:, 0]), ValueError, "history"), (dict(history=h, lengths=h[:1, 0]), ValueError, "lengths"),
            (dict(repetition=0.0), ValueError, "positive"), (dict(presence=float("nan")), ValueError, "finite"),
            (dict(repetition=torch.ones(3, device=cuda)), ValueError, "repetition"),
            (dict(presence=torch.ones(2)), RuntimeError, "GPU"),
            (dict(bias=x[:, 0, :3]), ValueError, "together"),
            (dict(bias=x[:, 0, :3].half(), bias_tokens=h[:, :3]), ValueError, "bias"),
            (dict(bias=x[:, 0, :3], bias_tokens=h[:, :2]), ValueError, "bias_tokens"),
            (dict(allowed=words.bool()), TypeError, "allowed"), (dict(allowed=words[:, :3]), ValueError, "allowed"),
            (dict(drafts=h[:, :3].long()), ValueError, "together"),
            (dict(drafts=h[:, :2].long(), parents=h[0, :3]), ValueError, "drafts"),
            (dict(drafts=h[:, :3].float(), parents=h[0, :3]), TypeError, "drafts"),
            (dict(drafts=h[:, :3].long(), parents=h[0, :2]), ValueError, "parents"),
            (dict(out=x[:, :2]), ValueError, "out"), (dict(out=x.half()), ValueError, "out"),
            (dict(out=x.clone().as_strided((2, 3, 100), (250, 50, 1))), ValueError, "overlap")):
        with pytest.raises(error, match=match):
            adjust_logits(x, **kw)
    with pytest.raises(ValueError, match="memory"):
        adjust_logits(x[:, :, :50], out=x[:, :, 25:75])
    with pytest.raises(RuntimeError, match="gradient"):
        adjust_logits(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="nodes"):
        big = torch.zeros((1, 257, 4), device=cuda)
        adjust_logits(big, drafts=torch.zeros((1, 257), dtype=torch.int64, device=cuda),
                      parents=torch.zeros(257, dtype=torch.int32, device=cuda))


def test_long_histories_and_lists(cuda):
    """Histories and lists on both sides of 2^15, where counts and places share a word."""
    for L, biases in ((32767, 5), (32768, 5), (40000, 70), (100, 32767), (100, 32768)):
        a = setup(2, 1, 5000, L, "fp32", biases=biases)
        a["history"][0] = 4999
        a["lengths"][0], a["prompts"][0] = L, 0
        check(a, call(a, cuda), "fp32")
