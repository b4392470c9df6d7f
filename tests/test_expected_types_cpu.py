"""What a refused tensor should have been is said in torch's names of types."""
import pytest
import torch

import lutmac_amd as L
from lutmac_amd import kv8


def z(*s, dtype=torch.float32):
    return torch.zeros(*s, dtype=dtype)


I32 = torch.int32


def pages():
    return kv8.KvPages(z(3, 4, dtype=I32), z(3, dtype=I32), z(9, dtype=I32), z(1, dtype=I32))


@pytest.mark.parametrize("call,said", [
    (lambda: L.linear_i8(z(2, 200), z(130, 208), z(130)), "expected int8 [rows, cols]"),
    (lambda: L.linear_f8(z(2, 200), z(130, 208), z(2, 2)), "expected float8_e4m3fn [rows, cols]"),
    (lambda: kv8.rotate(z(5, 4, 64), None, z(4, dtype=I32), z(9, 32, 2)), "expected contiguous int32 [5]"),
    (lambda: pages().extend(z(3, dtype=I32), z(8, dtype=I32), slots=z(8, dtype=I32)), "expected contiguous int64 [8]"),
    (lambda: L.verify_drafts(z(6, 50), z(6, dtype=I32), z(3, dtype=I32), z(6, 3)), "expected contiguous float32 [6, 2]"),
], ids=["linear_i8", "linear_f8", "rotate", "extend", "verify_drafts"])
def test_expected_types(call, said):
    with pytest.raises(ValueError) as e:
        call()
    assert said in str(e.value)
