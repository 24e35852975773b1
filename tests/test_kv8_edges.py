"""The 8-bit key/value cache on the CPU: what the kernels' reports name."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "slopllm_b200", "csrc")


def test_reports_name_one_kernel():
    """Numbers of failed self-checks and of expired waits in the 8-bit cache's kernels are no other kernel's, and are written by name."""
    text = {os.path.basename(f): open(f).read() for f in glob.glob(os.path.join(CSRC, "*.cu*"))}
    own = dict(re.findall(r"(KV8_(?:SITE|WAIT)_\w+) = (\d+)", text["kv8.cuh"]))
    sites, waits = ([int(v) for k, v in own.items() if k.startswith(f"KV8_{what}")] for what in ("SITE", "WAIT"))
    assert len(set(sites)) == 4 and len(set(waits)) == 2
    used = {"site": {}, "wait": {}}
    for name, source in text.items():
        for what, pattern in (("site", r"(?:guard_ok|kv8_slot)\(\s*[\w.>-]+(?:\([^()]*\))?,\s*(\d+)\s*,"), ("wait", r"atomicExch\([^;]*?,\s*(\d+)\)")):
            for number in re.findall(pattern, source):
                used[what].setdefault(int(number), set()).add(name)
    assert used["site"] and used["wait"]
    assert not set(sites) & set(used["site"]) and not set(waits) & set(used["wait"])
    assert not any(name.startswith("kv8") for names in (*used["site"].values(), *used["wait"].values()) for name in names)
