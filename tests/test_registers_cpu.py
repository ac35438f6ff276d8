"""What the compiler gives a kernel that hands registers around among its warps (no GPU needed)."""
import os
import re
import subprocess

from cobalt_b200 import build


def test_the_head_products_have_the_registers_that_they_hand_around(tmp_path):
    """A warp that asks for registers waits until the block has them: the kernel is launched only if it was built with HL_REGS a thread.  Nothing but the launch
    bounds asks the compiler for that number (a limit of its own excludes them), so another compiler shows here, not in a user's first loss."""
    header = open(os.path.join(build.CSRC, "head_loss.cuh")).read()
    want = int(re.search(r"HL_REGS = (\d+)", header).group(1))
    source = tmp_path / "registers.cu"
    source.write_text(f'#include "{os.path.join(build.CSRC, "head_loss.cuh")}"\n')
    log = subprocess.run([build._nvcc(), *build.FLAGS, "-Xptxas", "-v", "-c", str(source), "-o", str(tmp_path / "registers.o")], capture_output=True, text=True, check=True).stderr
    used = re.search(r"Function properties for \S*head_product_kernel\S*\n.*\n.*Used (\d+) registers", log)
    assert used and int(used.group(1)) == want, log
