"""The burn-in's fp4 step: what it gates, publishes and shows, and that it runs on the device."""
import pytest

from kubernetes_amd.deviceplugin.burnin import BurnIn, BurnInResult


def _result(**kw):
    return BurnInResult(ok=False, tflops=1400.0, hbm_gbps=6000.0, mfma_rel_err=1e-4, fp8_tflops=2800.0, fp8_rel_err=1e-5, **kw)


def test_judge():
    assert BurnIn().judge(_result()) == ""                                   # not asked for
    gate = BurnIn(min_fp4_tflops=2000.0)
    assert gate.judge(_result(fp4_tflops=4000.0, fp4_rel_err=1e-7)) == ""
    assert "fp4" in gate.judge(_result(fp4_tflops=1999.0, fp4_rel_err=1e-7))
    assert "fp4" in gate.judge(_result())                                    # not measured
    for err in (1.0, float("nan")):
        assert "relative error" in gate.judge(_result(fp4_tflops=4000.0, fp4_rel_err=err))


def test_step_runs_only_when_asked_for(monkeypatch):
    from kubernetes_amd.ops import hip_kernels as hk
    ran = []
    good = {"tflops": 5000.0, "max_rel_err": 0.0}
    monkeypatch.setattr(hk, "diag_vector_add", lambda dev, n: 0.0)
    monkeypatch.setattr(hk, "diag_mfma", lambda dev, size, iters: good)
    monkeypatch.setattr(hk, "diag_mfma_fp8", lambda dev, size, iters: good)
    monkeypatch.setattr(hk, "diag_mfma_fp4", lambda dev, size, iters: ran.append(dev) or good)
    monkeypatch.setattr(hk, "diag_hbm", lambda dev, nbytes, iters: {"GBps": 6000.0})
    r = BurnIn().run(3)
    assert r.ok and not ran and r.fp4_tflops == 0
    r = BurnIn(min_fp4_tflops=2000.0).run(3)
    assert r.ok and ran == [3] and r.fp4_tflops == 5000


def test_attribute(tmp_path):
    from kubernetes_amd.deviceplugin.amdgpu import ATTR_MFMA_FP4_TFLOPS, AMDGPUPlugin
    from kubernetes_amd.native import amdsmi
    smi = amdsmi.SMI(fixture=amdsmi.fixture_file(2, seed="fp4"))
    plugin = AMDGPUPlugin(str(tmp_path), smi=smi, health_interval=0, burn_in=BurnIn(min_fp4_tflops=2000.0))
    with_fp4, without = plugin.gpus
    plugin._burn = {with_fp4.device_id_str: _result(fp4_tflops=4321.9), without.device_id_str: _result()}
    assert plugin._device(with_fp4, smi.metrics(0), "Healthy").Attributes[ATTR_MFMA_FP4_TFLOPS] == "4321"
    assert ATTR_MFMA_FP4_TFLOPS not in plugin._device(without, smi.metrics(1), "Healthy").Attributes


def test_shown_by_describe_and_dashboard():
    from kubernetes_amd.addons import dashboard
    from kubernetes_amd.api import core
    from kubernetes_amd.kubectl.printers import describe
    attrs = {core.ATTR_INDEX: "0", "amd.com/burn-in": "passed", "amd.com/mfma-tflops": "1188",
             "amd.com/mfma-fp8-tflops": "2242", "amd.com/mfma-fp4-tflops": "4021", "amd.com/hbm-gbps": "6199"}
    node = {"kind": "Node", "metadata": {"name": "n"}, "spec": {},
            "status": {"extendedResources": {core.AMD_GPU: {"resources": {"g0": {"health": "Healthy", "attributes": attrs}}}}}}
    assert "(bf16 1188 / fp8 2242 / fp4 4021 TF/s, HBM 6199 GB/s)" in describe(node)
    device = {"id": "g0", "health": "Healthy", "hive": "", "numa": "", "partition": "SPX", "socket": "", "burn_in": "passed",
              "tflops": "1188", "fp8_tflops": "2242", "fp4_tflops": "4021", "pod": ""}
    state = {"gpus": {"total": 1, "allocated": 0, "healthy": 1}, "pods": [], "warnings": [],
             "nodes": [{"name": "n", "ready": True, "unschedulable": False, "gpus": 1, "allocated": 0, "healthy": 1,
                        "devices": [device]}]}
    assert "<td>1188 / 2242 / fp4 4021</td>" in dashboard.render(state)
    device["fp4_tflops"] = ""
    assert "<td>1188 / 2242</td>" in dashboard.render(state)


def test_c_entry_refuses_sizes():
    from kubernetes_amd.ops import hip_kernels as hk
    try:
        hk.load()
    except hk.HIPError:
        pytest.skip("the library is not built")
    for size, iters in ((0, 1), (-32, 1), (33, 1), (64, 0)):
        with pytest.raises(hk.HIPError, match="multiple of 32"):
            hk.diag_mfma_fp4(0, size, iters)


@pytest.mark.gpu
@pytest.mark.parametrize("size,iters", [(32, 1), (96, 2), (544, 2), (2048, 3), (4096, 5)])
def test_diag_mfma_fp4(size, iters):
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from kubernetes_amd.ops import hip_kernels as hk
    r = hk.diag_mfma_fp4(0, size, iters)
    print(r)
    # each of `size` additions is off by 2^-23 of the sum of magnitudes at most; a wrong code or scale gives 1
    assert r["max_rel_err"] <= size * 2.0 ** -23 and r["tflops"] > (1000 if size == 4096 else 0)


@pytest.mark.gpu
def test_burn_in_with_fp4():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    r = BurnIn(min_fp4_tflops=2000.0).run(0)
    print(r)
    assert r.ok, r.reason
    assert r.fp4_tflops > 2000 and r.fp4_rel_err < 1e-4
