"""``out=`` of attend and qk_norm_rotate: the input itself, a part of its product, or refused."""
import pytest

import slime_amd

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def _draw(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Nq,Nk,Hq,Hkv,D", [(1, 65, 8, 8, 64), (2, 3000, 4, 1, 32), (77, 77, 4, 2, 16), (300, 2000, 2, 2, 128),
                                            (513, 513, 8, 8, 64)])
def test_the_queries_themselves(dtype, Nq, Nk, Hq, Hkv, D):
    """Few rows and many, walks of one part and of several: the bits of a call with an output of its own."""
    q, k, v = _draw((2, Nq, Hq, D), dtype, 1), _draw((2, Nk, Hkv, D), dtype, 2), _draw((2, Nk, Hkv, D), dtype, 3)
    lengths = torch.tensor([Nk, Nk // 2], dtype=torch.int32, device="cuda")
    want = slime_amd.attend(q, k, v, lengths=lengths, causal=True)
    out, lse = slime_amd.attend(q, k, v, lengths=lengths, causal=True, out=q)
    assert out.data_ptr() == q.data_ptr() and torch.equal(q, want[0]) and torch.equal(lse, want[1])


def test_a_part_of_one_product():
    x = _draw((2, 40, 16, 32), torch.bfloat16)
    q, k, v, y = x[:, :, :4], x[:, :, 4:8], x[:, :, 8:12], x[:, :, 12:]
    want, _ = slime_amd.attend(q, k, v)
    slime_amd.attend(q, k, v, out=y)
    assert torch.equal(y, want)
    wq, wk = torch.ones(32, device="cuda"), torch.full((32,), 0.5, device="cuda")
    pos = torch.arange(40, dtype=torch.int32, device="cuda").view(1, 40, 1).expand(2, -1, -1)
    args = (wq, wk, pos, slime_amd.rotation_freqs(32))
    want = slime_amd.qk_norm_rotate(q, k, *args)
    keys = x[:, :, 8:12]
    slime_amd.qk_norm_rotate(q, k, *args, out=(q, keys))
    assert torch.equal(q, want[0]) and torch.equal(keys, want[1])


def test_outputs_in_other_memory_of_the_call_are_refused():
    x = _draw((2, 40, 12, 32), torch.float32)
    q, k, v = x[:, :, :4], x[:, :, 4:8], x[:, :, 8:]
    before = x.clone()
    for out, name in ((k, "k"), (v, "v"), (x[:, :, 2:6], "q"), (x[:, :, 7:11], "k")):
        with pytest.raises(ValueError, match=f"out lies in the memory of {name}"):
            slime_amd.attend(q, k, v, out=out)
        with pytest.raises(ValueError, match="out lies in the memory of"):
            slime_amd.attend(q, k, v, out=out, stream=torch.cuda.Stream())
    own = torch.zeros(2, 40, 4, 32, device="cuda")
    mask = own.view(torch.uint8).view(-1)[:80].view(2, 40)
    with pytest.raises(ValueError, match="out lies in the memory of alive"):
        slime_amd.attend(q, k, v, out=own, alive=mask)
    wq, wk = own.view(-1)[:32], torch.ones(32, device="cuda")
    pos = torch.zeros(2, 40, 1, dtype=torch.int32, device="cuda")
    freqs = slime_amd.rotation_freqs(32)
    other = torch.empty_like(own)
    for out, name in (((k, other), r"out\[0\] lies in the memory of k"), ((other, q), r"out\[1\] lies in the memory of q"),
                      ((other, other), r"out\[1\] lies in the memory of out\[0\]"),
                      ((own, other), r"out\[0\] lies in the memory of wq")):
        with pytest.raises(ValueError, match=name):
            slime_amd.qk_norm_rotate(q, k, wq, wk, pos, freqs, out=out)
    torch.cuda.synchronize()
    assert torch.equal(x, before)
