"""Which kernels of the paged cache's attention the library holds (its exported symbols, no GPU): those that a call can reach."""
import pytest

NAMES = {"f16": "DF16_", "bf16": "DF16b", "e4m3": "h"}
PAIRS = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "e4m3"), ("f16", "e4m3")]


def kernel(name, q, cache, *more):
    return f"_ZN2qm{len(name)}{name}I{NAMES[q]}{NAMES[cache]}{''.join(more)}EEvNS_8AttnArgsE"


@pytest.mark.parametrize("q,cache", PAIRS)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_variants(qm, q, cache, D):
    """Weights in one part for 16-bit results of the matrix pipe's type; f16 behind an 8-bit cache in two; f32 in two of f16, three of bf16. Row tiles
    of 16 to 64 (heads of up to 64), 32 (128) or 16; large ones of 64 and 128 rows, of 64 alone for heads beyond 128, 128 alone behind
    8-bit caches of shorter ones."""
    lib = qm.load_library()
    parts = {("bf16", "bf16"): {1, 3}, ("f16", "f16"): {1, 2}, ("bf16", "e4m3"): {1, 3}, ("f16", "e4m3"): {2, 3}}[q, cache]
    few = {64: {1, 2, 4}, 128: {1, 2}, 256: {1}}[D]
    many = {1} if D == 256 else {2} if cache == "e4m3" else {1, 2}
    for full in (0, 1):
        for mt in (1, 2, 3, 4):
            for n in (1, 2, 3):
                at = f"Li{D}E", f"Lb{full}E", f"Li{mt}E", f"Li{n}E"
                for chosen in (0, 1):
                    assert hasattr(lib, kernel("attn_kernel", q, cache, *at, f"Lb{chosen}E")) == (mt in few and n in parts), (full, mt, n)
                assert hasattr(lib, kernel("attn_tile_kernel", q, cache, *at)) == (mt in many and n in parts), (full, mt, n)
