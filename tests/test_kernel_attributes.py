"""What a kernel is allowed (shared memory, cluster sizes) belongs to a device: it is asked for on every device, not once per process."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tinyflow_b200", "csrc")


def test_attributes_are_set_on_every_device():
    found = []
    for name in sorted(os.listdir(CSRC)):
        code = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        for m in re.finditer(r"cudaFuncSetAttribute", code):
            # the statements around it: a flag or a static that outlives the call says that a process does it once
            around = code[max(0, m.start() - 220):m.start()]
            each_call = re.search(r"TF_CUDA\(\s*$", around) and not re.search(r"done\w*\s*(\[[^\]]*\])?\s*\)", around)
            if not each_call and "once_per_device" not in around:
                found.append((name, code[m.start():m.start() + 60]))
    assert not found
