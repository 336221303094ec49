"""strasgpt_k_lora above 512 tokens, whose kernel is another one than the few tokens': the
forms of a call that test_lora.py makes with few. Tolerances are test_lora's.
"""
import pytest
import test_lora as lora

F32, BF16 = lora.F32, lora.BF16
STORE, ADD, SWIGLU = lora.STORE, lora.ADD, lora.SWIGLU


def inputs(torch, m, k, n, r, d, type_, seed):
    """Mixed adapters at both ends; runs between them, whose borders lie inside tiles."""
    x, a, b, adapter, scale, base = lora.inputs(torch, m, k, n, r, d, type_, seed)
    at = 40
    for length, of in ((130, 0), (1, d - 1), (31, -1), (200, 1), (33, 0), (150, d - 1)):
        adapter[at:at + length] = of
        at += length
    return x, a, b, adapter, scale, base


def fits(got, want_err):
    want, err = want_err
    return ((got.double() - want).abs() <= err).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type_", [F32, BF16])
@pytest.mark.parametrize("epi", [STORE, ADD, SWIGLU])
@pytest.mark.parametrize("m,r,n", [(700, 16, 178), (700, 16, 182), (700, 72, 18), (1300, 72, 194),
                                   (2500, 64, 190), (700, 8, 192), (600, 8, 2)])
def test_entries_behind_the_rows_stay(cuda, type_, epi, m, r, n):
    """Rows of out on 16 bytes within wider ones and before other memory, which end
    anywhere within 16 bytes: all around them stays as it is, behind the last row too."""
    torch = cuda
    x, a, b, adapter, scale, base = inputs(torch, m, 264, n, r, 3, type_, m + n)
    outs = n // 2 if epi == SWIGLU else n
    ld = (outs + 7) // 8 * 8
    for wider in (ld, ld + 24):
        flat = torch.randn(m * wider + 64, device="cuda").to(x.dtype)
        before, part = flat.clone(), flat[:m * wider].view(m, wider)[:, :outs]
        want = lora.reference(torch, x, a, b, adapter, scale, base, part, epi, type_)
        assert lora.call(torch, x, a, b, adapter, scale, base, part, epi, type_) == 0
        assert fits(part, want)
        part.copy_(before[:m * wider].view(m, wider)[:, :outs])
        assert torch.equal(flat, before)
