"""The workspace of the SAE's gradient holds what its plan writes, without a GPU."""
import pytest

from streamtopk_sae import _capi


def part(N, d):
    """Codes of one feature that are summed at a time, of more than 8192."""
    n = 32 if N < 65536 else 64
    while n < 256 and 2 * (N // n) * d > 2 ** 25:
        n *= 2
    return n


@pytest.mark.parametrize("B,k,F,d,codes", [
    (4096, 64, 65536, 2048, 64), (1001, 33, 20000, 1032, 32), (8192, 64, 70, 4096, 128), (16384, 64, 70, 4096, 256),
    (131072, 64, 65536, 2048, 256), (300, 40, 5_000_000, 8, 32), (2101, 4, 30, 20008, 32)])
def test_workspace_holds_codes_bounds_and_partial_sums(B, k, F, d, codes):
    N = B * k
    assert part(N, d) == codes
    slots = 2 * (N // codes)            # lists longer than a part, and the full parts of them
    need = 4 * 4 * N                    # two buffers of keys and codes
    need += 4 * 2048 * -(-N // 1024)    # a count for each digit and tile
    need += 4 * (F + 1)                 # each feature's first code
    need += 24 * (N // 9 + N // codes)  # lists of more than 8 codes, and parts
    need += slots * (2 * 4 * d + 8)     # sums of parts, for both dictionaries, and who has arrived
    need += 4 * d * (1 + min(32, -(-B // 128)))
    got = _capi.sae_backward_workspace_bytes(B, k, F, d)
    assert need <= got <= need + 4 * -(-d // 128) + 20 * 256 + 4 * 2048 + 16
