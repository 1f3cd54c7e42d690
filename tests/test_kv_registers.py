"""The attention kernels that bring the cache to the LDS by load-to-LDS instructions count those by hand: nothing of an instance may lie in scratch memory, whose loads and
stores go through the same counter. Compiled to assembly, so without a device."""
import concurrent.futures
import os
import re
import tempfile

from tests.test_stream_loop_waits import _assembly

UNITS = ["kv_attention_rows.hip", "kv_attention_quads.hip", "kv_attention_prompts.hip"]


def test_no_scratch():
    with tempfile.TemporaryDirectory() as d, concurrent.futures.ThreadPoolExecutor(len(UNITS)) as pool:
        units = list(pool.map(lambda u: _assembly(u, os.path.join(d, u + ".s")), UNITS))
    for unit, lines in zip(UNITS, units):
        sizes, name = {}, None
        for line in lines:
            if m := re.match(r"\s*\.amdhsa_kernel (\S+)", line):
                name = m.group(1)
            elif m := re.match(r"\s*\.amdhsa_private_segment_fixed_size (\d+)", line):
                sizes[name] = int(m.group(1))
        assert len(sizes) >= 15 and not any(sizes.values()), (unit, {k: v for k, v in sizes.items() if v})
        assert not any("scratch_load" in line or "scratch_store" in line for line in lines), unit
