"""Which kernel prompts over the 8-bit cache take, by the times that both sides measured (us, streamed / not)."""
import pytest

from picolm_b200.ops.kv8 import kv8_streams


@pytest.mark.parametrize("walks,rows,keys,hd,streamed", [
    (8, 128, 8000, 96, True),            # 32 / 279
    (8, 256, 8000, 80, True),            # 45 / 270
    (2, 256, 8000, 256, True),           # 35 / 563
    (8, 128, 1000, 32, True),            # 12 / 37
    (128, 128, 3000, 80, True),          # 80 / 151
    (128, 128, 500, 96, False),          # 45 / 35
    (512, 256, 1000, 80, False),         # 248 / 177
    (8, 264, 8000, 96, False),           # (more rows than the streaming kernel is given)
    (512, 64, 1000, 96, True),           # 86 / 93
    (32, 32, 3000, 128, True),           # 23 / 35
    (80, 32, 2000, 128, False),          # 40 / 27
    (512, 32, 1000, 128, False),         # 67 / 55
    (8, 32, 1000, 64, True),             # 14 / 15
    (128, 64, 1000, 64, False),          # 25 / 16
])
def test_the_faster_one(walks, rows, keys, hd, streamed):
    assert kv8_streams(walks, rows, keys, hd) is streamed
