"""What the library exports: the C entry points and names of its own namespace, nothing that another library could define too."""
import subprocess

from pufferlean_amd import _lib as L

OTHERS = {"cuda_lstm_ppo_grad_batch", "g_mgLoss", "g_mgLossOn"}  # resolved by name by the reference's own objects


def test_no_name_outside_the_prefix():
    L.lib()
    out = subprocess.run(["nm", "-D", "--defined-only", str(L.LIB_PATH)], capture_output=True, text=True, check=True).stdout
    names = [line.split()[-1] for line in out.splitlines() if line.split()[-2] in "TtDBR"]
    assert "ph_version" in names
    strange = [n for n in names if not n.startswith(("ph_", "_ZN2ph", "_ZNK2ph", "__hip_")) and n not in OTHERS]
    assert not strange, strange
