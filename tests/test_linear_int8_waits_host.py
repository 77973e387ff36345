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


def test_no_columns_are_held_in_a_wait_for_other_blocks():
    """A part of K gives its tensor memory back before it waits for the other parts: a
    pair of blocks that waits for those columns may hold what the other parts wait for."""
    body = kernel("narrow_kernel")
    frees = re.search(r"auto (\w+) = \[&\]\(\) \{[^}]*__syncthreads\(\);[^}]*tmem_dealloc\(", body, re.S)
    parts = body[body.index("if (split == 1)"):].split("} else {", 1)[1]
    first = parts.index("cluster_sync_all();")
    assert frees and f"{frees.group(1)}();" in parts[:first]
    assert "tmem_ld" not in parts[first:] and "load(" not in parts[first:]
    assert body.count("tmem_dealloc(") == 1 and body.count(f"{frees.group(1)}();") == 2


def test_copies_in_flight_land_after_any_failure():
    """Whichever role gives up, a block's memory is not released before its copies
    have landed or a limit has passed: the wait stands behind all roles."""
    body = kernel("narrow_kernel")
    end = body[body.index("auto free_columns"):body.index("if (split == 1)")]
    assert re.search(r"__syncthreads\(\);.*if \(threadIdx.x == 0 && \*abort_flag\)\s*for \(int j = [^;]*; j < issued; \+\+j\)"
                     r"\s*mbar_wait_ns\(&full\[j % stages\]", end, re.S)
    body = kernel("wide_kernel")
    end = body[body.rindex("__syncthreads();"):]
    assert re.search(r"if \(warp == 0 && \*abort_flag\) \{.*globaltimer_ns\(\) - t0 < 1000000ull.*cluster_sync_all\(\);", end, re.S)
