"""What the 8-bit linear layer's kernels do when a bounded wait runs out. No
test makes one run out on a GPU: the steps are read from the source."""
import pathlib
import re

from wide_compiler import ops

SRC = (pathlib.Path(ops.__file__).resolve().parents[1] / "csrc" / "linear_int8.cu").read_text()


def kernel(name):
    body = SRC[SRC.index(name + "("):]
    return body[:body.index("\n}\n")]


def test_the_last_wait_of_narrow_tiles_is_reported():
    """Accumulators that are not finished in time are neither stored nor passed over in silence."""
    body = kernel("narrow_kernel")
    after = body[body.index("mbar_wait(&tfull"):]
    report = re.search(r"if \(!ok\) \{(.*?)\}", after, re.S)
    assert report and "raise_device_error" in report.group(1) and "*abort_flag = 1" in report.group(1)
    epilogue = after[report.end():]
    whole, parts = epilogue[epilogue.index("if (split == 1)"):].split("} else {", 1)
    assert re.search(r"for \([^;]*; ok && [^;]*;", whole), "tiles of one CTA are stored without a look at the wait"
    adding = parts[parts.index("cluster_sync_all();"):parts.rindex("cluster_sync_all();")]
    calls = re.findall(r"if \((.*)\) add_parts<", adding)
    assert len(calls) == adding.count("add_parts<") == 3
    assert all(c.startswith("ok") for c in calls), "parts are added without a look at the wait"
