"""Which kernels of the q/k norm + rotation the library holds (its exported symbols, no GPU): those that a call can reach."""
import pytest

NAMES = {"f32": "f", "f16": "DF16_", "bf16": "DF16b"}


def kernel(x, out, v, u, b):
    return f"_ZN2qm19qk_norm_rope_kernelI{NAMES[x]}{NAMES[out]}Li{v}ELi{u}ELi{b}EEEvNS_8RopeArgsEii"


@pytest.mark.parametrize("x", NAMES)
@pytest.mark.parametrize("out", NAMES)
def test_eight_values_at_a_time_are_of_16_bits(qm, x, out):
    """By the element, heads of up to 128 and longer ones; four at a time; eight where both sides are of 16 bits."""
    lib = qm.load_library()
    for v, u, b, there in ((1, 1, 1, True), (1, 4, 1, True), (4, 1, 2, True), (8, 1, 2, x != "f32" and out != "f32")):
        assert hasattr(lib, kernel(x, out, v, u, b)) == there, (x, out, v)
