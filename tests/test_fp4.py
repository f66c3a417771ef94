"""The plain restatement of rows in microscaled 4-bit floating point against itself, and the refusals that need no GPU."""

import pytest
import torch

import plain_fp4 as plain


def test_rounding_by_hand():
    x = torch.tensor([[7.0, 6.9, 5.0, 2.5, -0.25, 0.26, -3.5, 1.75] + [0.0] * 24, [7.01, 5.0] + [0.0] * 30])
    assert plain.scale_exponents(x)[:, 0].tolist() == [0, 1]
    assert plain.rounded(x)[0, :8].tolist() == [6.0, 6.0, 4.0, 2.0, -0.0, 0.5, -4.0, 2.0]
    assert plain.rounded(x)[1, :2].tolist() == [8.0, 4.0]


def test_reading_by_hand():
    codes = torch.zeros(130, 80, dtype=torch.uint8)
    scales = torch.zeros(2, 2, 512, dtype=torch.uint8)
    codes[129, 64] = 0x9F  # values 128 (-6) and 129 (-0.5) of the last row: block 4, tile (1, 1)
    scales[1, 1, 16] = 130
    v, byte = plain.read(codes, scales, 160)
    assert v[129, 128:130].tolist() == [-48.0, -4.0] and int(byte[129, 4]) == 130 and int(v.count_nonzero()) == 2


def test_tensors_off_the_gpu_are_refused():
    from qwen3_from_scratch_b200.kernels import ops
    r = ops.fp4_rows(2, 64, "cpu")
    assert r.rows == 2 and r.codes.shape == (2, 32) and r.scales.shape == (1, 1, 512) and r.first(1).rows == 1
    with pytest.raises(ops.KernelError, match="GPU only"):
        ops.fp4_quantise(torch.zeros(2, 64), r)
    with pytest.raises(ops.KernelError, match="GPU only"):
        ops.fp4_product(r, r, torch.zeros(2, 2), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ops.KernelSizeError):
        ops.fp4_rows(-1, 64, "cpu")


@pytest.mark.parametrize("wide", [torch.int16, torch.int32, torch.int64])
def test_bytes_in_a_wider_integer_type_are_read_as_bytes(wide):
    from qwen3_from_scratch_b200.kernels import ops
    codes = torch.arange(256, dtype=torch.uint8).view(8, 32)
    scales = (torch.arange(512) % 256).to(torch.uint8).view(1, 1, 512)
    for c, s in ((codes.to(wide), scales), (codes, scales.to(wide)), (codes.to(wide), scales.to(wide))):
        r = ops._fp4_bytes(ops.Fp4Rows(c, s, 64))
        assert r.codes.dtype is r.scales.dtype is torch.uint8 and r.width == 64
        assert torch.equal(r.codes, codes) and torch.equal(r.scales, scales)
    own = ops.Fp4Rows(codes, scales, 64)
    assert ops._fp4_bytes(own) is own
    other = ops.Fp4Rows(codes.float(), scales, 64)
    assert ops._fp4_bytes(other).codes.dtype is torch.float32


def test_the_command_line_does_not_drop_the_option(tmp_path):
    from qwen3_from_scratch_b200.cli import main
    config = tmp_path / "batch.yaml"
    config.write_text("models: []\n")
    with pytest.raises(SystemExit, match="--feed-forward-weights"):
        main(["generate", "--config-path", str(config), "--model-name", "a", "--feed-forward-weights", "fp4", "--prompt-ids", "1 2"])


def test_an_unknown_form_is_refused():
    from qwen3_from_scratch_b200.kernels import ops
    assert [ops._fp4_form("p", f) for f in (None, "few", "pair384")] == [0, 1, 384]
    with pytest.raises(ops.KernelError, match="no form 'pair128'"):
        ops._fp4_form("p", "pair128")
