"""The training operators' sizes on devices of different compute units, without
a GPU: a workspace is sized for the device that the call runs on."""

import pytest


class _Devices:
    """A library whose plan counts the current device's compute units."""

    current = 0

    def pdh_linear_xent_workspace(self, *args):
        return 1024 * (self.current + 1)


def test_the_heads_workspace_is_the_current_devices(monkeypatch):
    torch = pytest.importorskip("torch")
    from pdum_dsl_amd import _lib
    from pdum_dsl_amd import kernels as K

    devices = _Devices()
    monkeypatch.setattr(_lib, "lib", lambda: devices)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: devices.current)
    args = (0, 0, 12345, 768, 6789, 768, 768, 1, 1)  # sizes that nothing else asks for
    for devices.current in (0, 1, 0, 1):
        assert K._head_workspace(*args) == 1024 * (devices.current + 1)
