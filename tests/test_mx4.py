"""What rows in 4 bits are made of, and what is refused before any kernel runs."""
import pytest
import torch

import mx4_util as mx


def test_layout_of_codes_and_scales():
    from cuca_b200.kernels import ops
    q = ops.Mx4Matrix.empty(300, 200, "cpu")
    assert q.shape == (300, 200) and q.codes.shape == (300, 128) and q.scales.shape == (3, 2, 32, 4, 4)
    assert q.nbytes == 300 * 128 + 3 * 2 * 512 and q.device.type == "cpu"
    q.codes.zero_()
    code, byte = torch.randint(0, 16, (300, 7, 32)), torch.randint(0, 256, (300, 7))
    flat = code.flatten(1)
    for i, (low, high) in enumerate(((0, 2), (4, 6), (1, 3), (5, 7))):
        q.codes[:, i:112:4] = (flat[:, low::8] + 16 * flat[:, high::8]).to(torch.uint8)
    for r in range(300):
        for b in range(7):
            q.scales[r // 128, b // 4, r % 32, r % 128 // 32, b % 4] = byte[r, b]
    got = mx.unpack(q)
    assert torch.equal(got[0], code) and torch.equal(got[1], byte)


@pytest.mark.parametrize("rows,cols,codes,scales", [
    (4, 0, (4, 0), (1, 0, 32, 4, 4)), (4, 64, (4, 32), (1, 1, 32, 4, 4)), (4, 64, (3, 64), (1, 1, 32, 4, 4)),
    (4, 64, (4, 64), (1, 2, 32, 4, 4)), (129, 64, (129, 64), (1, 1, 32, 4, 4)), (4, 64, (4, 64), (512,))])
def test_memory_of_another_shape_is_refused(rows, cols, codes, scales):
    from cuca_b200.kernels import library, ops
    with pytest.raises(library.KernelError):
        ops.Mx4Matrix(rows, cols, torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8))


def test_memory_of_another_type_or_with_gaps_is_refused():
    from cuca_b200.kernels import library, ops
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8)
    ops.Mx4Matrix(4, 64, codes, scales)
    for c, s in ((codes.to(torch.int8), scales), (codes, scales.float()), (torch.zeros(4, 128, dtype=torch.uint8)[:, ::2], scales),
                 (codes, scales.transpose(2, 3).contiguous().transpose(2, 3).expand(1, 1, 32, 4, 4).flip(4)[..., ::1].transpose(3, 4))):
        with pytest.raises(library.KernelError):
            ops.Mx4Matrix(4, 64, c, s)


def test_there_is_no_cpu_path():
    from cuca_b200.kernels import library, ops
    q = ops.Mx4Matrix.empty(4, 64, "cpu")
    for call in (lambda: ops.mx4_quantise(torch.zeros(4, 64)), lambda: ops.mx4_values(q, torch.zeros(4, 64)),
                 lambda: ops.gemm_mx4(torch.zeros(2, 64, dtype=torch.bfloat16), q, torch.zeros(2, 4))):
        with pytest.raises(library.KernelError):
            call()


def test_rows_that_overlap_are_refused_at_the_c_entry():
    """The host's checks come before any launch: no kernel runs here."""
    from cuca_b200.kernels import library, ops
    lib = library.load()
    at = 1 << 20
    for kind, lda, ldo in ((1, 63, 10), (0, 63, 10), (1, 64, 9), (2, 0, 9)):
        call = ops._MX4_GEMM.pack(at, at, lda, kind, at, at, 0, at, ldo, 1, 0, 20, 10, 64, 0, at, 0, 0)
        assert lib.cuca_gemm_mx4(call) != 0 and b"overlap" in lib.cuca_last_error()
    call = ops._MX4_ROWS.pack(at, 63, 0, at, at, 2, 64, 0)
    for entry in (lib.cuca_mx4_quantise, lib.cuca_mx4_values):
        assert entry(call) != 0 and b"overlap" in lib.cuca_last_error()


def test_the_formula_against_a_search():
    """The nearest of the sixteen values for every block, found by trying all of them."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(20, 70, generator=g) * torch.exp2(torch.randint(-30, 30, (20, 1), generator=g).float())
    code, byte = mx.quantise(x)
    got = mx.values(code, byte, 70)
    table = torch.tensor(mx.MAGNITUDES, dtype=torch.float64)
    for r in range(20):
        for b in range(3):
            v = x[r, 32 * b:32 * b + 32].double()
            power = 2.0 ** (int(byte[r, b]) - 127)
            assert 4 * power <= v.abs().max() < 8 * power
            best = (v.abs()[:, None] - table * power).abs().min(1).values
            assert torch.equal((v - got[r, 32 * b:32 * b + 32]).abs(), best)
