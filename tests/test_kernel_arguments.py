"""CPU: the explicit arguments of every optimiser kernel, as compiled, keep to the 4 KB that csrc/optim.hip claims for them."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_optimiser_kernels_keep_to_4_kb_of_arguments(tmp_path):
    out = str(tmp_path / "optim.s")
    subprocess.check_call([os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), "--offload-arch=gfx950", "-O1", "-std=c++17", "--cuda-device-only", "-S",
                           os.path.join(ROOT, "nndetection_amd", "csrc", "optim.hip"), "-o", out], stderr=subprocess.DEVNULL)
    text = open(out).read()
    meta = text[text.index("amdhsa.kernels:"):text.index("amdhsa.target:")]
    sizes = {}
    for kernel in meta.split("\n  - ")[1:]:
        name = re.search(r"\.symbol:\s+'?(\w+)\.kd", kernel).group(1)
        args = kernel[kernel.index(".args:"):]
        end = [int(re.search(r"\.offset:\s+(\d+)", a).group(1)) + int(re.search(r"\.size:\s+(\d+)", a).group(1))
               for a in re.split(r"\n\s+- ", args) if ".value_kind" in a and "hidden_" not in a]
        sizes[name] = max(end)
    assert len(sizes) >= 40 and max(sizes.values()) > 4000
    assert {k: v for k, v in sizes.items() if v > 4096} == {}
