"""A tensor's number is checked on the host."""
import pytest


@pytest.mark.parametrize("number,rc", [(-1, 1), (1 << 29, 1), (0, 0), ((1 << 29) - 1, 0)])
def test_tensor_numbers(number, rc):
    from dnanet_amd import hip
    row = (hip.DnAdamwTensor * 2)(hip.DnAdamwTensor(4096, 4096, 0, 0, 0.0, 0, 0, 0), hip.DnAdamwTensor(4096, 4096, 8 if rc else 0, 0, 0.0, 0, 0, number))
    assert hip.lib.dn_adamw_step(row, 2, 4096, 4096, 4096, 4096, 8, 1e-3, 0.9, 0.999, 1e-8, 1, 0, None, 0, None) == rc
    if rc:
        assert b"number" in hip.lib.dn_last_error()
    assert hip.lib.dn_grad_norm_workspace_bytes(row, 2) > 0, "the norm does not ask for it"
