"""shared_decode of a step without rows: its sequences have contexts, and neither
query nor output has a byte."""

import numpy as np
import pytest

from swiftllm_amd._hip import DeviceArray, synchronize
from test_gpu_shared_decode import Shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tight", [False, True])
@pytest.mark.parametrize("off", [[0, 0, 0, 0, 0], [0, 1, 2, 3, 4]])
def test_no_rows(dev, tight, off):
    s = Shared(np.random.default_rng(1), [(160, [170, 180, 190, 200])], 8, 2, 64, "f16", tight=tight)
    s.d["q"] = DeviceArray((0,), np.uint16)
    s.run_plan()
    s.ws.fill_byte(0x5A)
    s.run_decode(query_offsets=DeviceArray.from_numpy(np.array(off, np.int32)), num_tokens=0)
    synchronize()
    assert (s.out.numpy() == 0x7F7F).all() and (s.ws.numpy() == 0x5A).all()
