"""Weight.codes_i8 on a given stream."""
import pytest
import torch

import lutmac_amd as L

pytestmark = pytest.mark.gpu


def test_codes_on_a_given_stream_own_what_they_write(cuda):
    """The codes and scales of a call on a given stream are that stream's memory: not
    what another stream has just freed, with work on it perhaps under way."""
    rows, cols = 1024, 4096
    planes, scales, _ = L.quantize(L.FMT_INT8, L.synth_normal(3, 0, rows, cols, 0.02), cols)
    w = L.Weight.from_planes(L.FMT_INT8, planes, scales, rows, cols, 0)
    first = [t.clone() for t in w.codes_i8()]
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    freed = [torch.empty(rows, cols, dtype=torch.int8, device="cuda"), torch.empty(rows, dtype=torch.float32, device="cuda")]
    places = [t.data_ptr() for t in freed]
    del freed
    got = w.codes_i8(stream=other)
    torch.cuda.synchronize()
    for t, place, want in zip(got, places, first):
        assert t.data_ptr() != place
        assert torch.equal(t, want)
