"""The counter-based generator against the known answers that its authors
publish for Philox4x32 with seven rounds."""

import pytest
import torch

from wap_amd.ops.dropout import _words

ONES = 0xFFFFFFFF


@pytest.mark.parametrize("counter,key,want", [
    ([0, 0, 0, 0], [0, 0], [0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48]),
    ([ONES] * 4, [ONES] * 2, [0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     [0x4DFCCABA, 0x190A87F0, 0xC47362BA, 0xB6B5242A]),
])
def test_known_answers(counter, key, want):
    assert _words(*(torch.tensor([v]) for v in counter + key)).tolist() == [want]
