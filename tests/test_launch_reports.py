"""What a launch reports is what ran."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
import kernels  # noqa: E402


def block_scaled_info(lengths, n, k):
    rows, experts = sum(lengths), len(lengths)
    ones = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device="cuda").fill_(127).view(torch.float8_e8m0fnu)  # noqa: E731
    a = torch.zeros((rows, k), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    b = torch.zeros((experts, n, k), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    ends = torch.tensor(lengths, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    kernels.launch_block_scaled_mm(a, ones(rows, -(-k // 128)), b, ones(experts, -(-n // 128), -(-k // 128)), ends)
    return kernels.last_block_scaled_info()


@pytest.mark.gpu
def test_block_scaled_grid_counts_the_ctas():
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    pair = block_scaled_info([900, 900], 2048, 256)  # 10 row blocks x 8: 80 tiles of two CTAs
    assert pair["path"] == "tcgen05_tma_pair"
    assert pair["grid"] % 2 == 0 and 80 < pair["grid"] <= sms  # fewer pairs than tiles
    one = block_scaled_info([40, 50], 264, 256)  # 2 row blocks x 3, one CTA each
    assert one["path"] == "tcgen05_tma" and one["grid"] == 6
    split = block_scaled_info([64], 264, 4096)  # 3 tiles, each shared by eight CTAs
    assert split["path"] == "tcgen05_tma" and split["grid"] == 24
    few = block_scaled_info([3, 2], 40, 256)  # 16 weight rows a CTA
    assert few["path"] == "warp_mma" and few["grid"] == 6
    kernels.check_device_errors()
