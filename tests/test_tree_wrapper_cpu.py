"""What the torch wrapper of the drafted-token step (opworks_b200/tree.py) decides on the host: nothing here launches."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")


def test_record_bytes_through_the_binding():
    import opworks_b200

    ops = opworks_b200.ops_lib()
    assert ops.kv_quant_record_bytes(64) == 32 * 64 + 128 and ops.kv_quant_record_bytes(128) == 32 * 128 + 128
    assert ops.reduction_workspace_size(1 << 20) > 0
    with pytest.raises(ValueError, match="head_dim"):
        ops.kv_quant_record_bytes(80)
