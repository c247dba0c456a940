"""install(layer_norm=True, rms_norm=True) rebinds the norms' Functions at the places where an installed liger_kernel binds them,
and the default install leaves them alone."""

import sys
import types

_SITES = {"LigerLayerNormFunction": ["liger_kernel.ops", "liger_kernel.transformers.functional", "liger_kernel.transformers.layer_norm"],
          "LigerRMSNormFunction": ["liger_kernel.ops", "liger_kernel.transformers.functional", "liger_kernel.transformers.rms_norm"]}


def _fake(monkeypatch):
    names = {"liger_kernel", "liger_kernel.ops", "liger_kernel.transformers", "liger_kernel.transformers.functional",
             "liger_kernel.transformers.fused_linear_cross_entropy", *sum(_SITES.values(), [])}
    mods = {n: types.ModuleType(n) for n in names}
    for n, m in mods.items():
        monkeypatch.setitem(sys.modules, n, m)
    return mods


def test_install_on_request_rebinds_the_norms(monkeypatch):
    import liger_kernel_b200 as lk

    mods = _fake(monkeypatch)
    assert lk.install() is True
    assert not any(hasattr(mods[site], symbol) for symbol, sites in _SITES.items() for site in sites)
    assert lk.install(layer_norm=True, rms_norm=True) is True
    for symbol, sites in _SITES.items():
        for site in sites:
            assert getattr(mods[site], symbol) is getattr(lk, symbol)


def test_install_without_that_module_is_reported(monkeypatch):
    import liger_kernel_b200 as lk

    _fake(monkeypatch)
    monkeypatch.setitem(sys.modules, "liger_kernel.transformers.rms_norm", None)       # import raises ImportError
    assert lk.install(rms_norm=True) is False
