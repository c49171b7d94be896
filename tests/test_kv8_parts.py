"""An engine asks every part that keeps keys and values whether it takes a cache in 8 bits, also parts that do not say."""
from types import SimpleNamespace

import pytest
import torch

from picolm_b200.cache import CacheSpec
from picolm_b200.engine import Engine


class Foreign:
    """A part of a program's own, not derived from this package's."""
    family, kind = "mixer", "its own"

    def cache_spec(self):
        return CacheSpec.kv(2, 64, None)


def test_a_part_that_does_not_say_is_refused():
    block = SimpleNamespace(parts=lambda: [("mixer", Foreign())])
    model = SimpleNamespace(loaded=True, runtime=SimpleNamespace(dtype=torch.bfloat16, device="cpu"), spec=SimpleNamespace(max_positions=256), blocks=[block])
    with pytest.raises(ValueError, match="takes_kv8"):
        Engine(model, 256, cache_type="e4m3")
