"""The autograd nodes of the experts' operators load on a machine without a GPU, by the first call that needs them."""
import os
import subprocess
import sys

PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jax-gptq_amd")


def test_nodes_load_and_take_the_librarys_entry_points():
    from jax_gptq_amd import _native as N
    nodes = N.load_torch()
    assert nodes is N.load_torch() and all(hasattr(nodes, f) for f in ("sort", "gather", "combine", "matmul"))


def test_importing_the_package_needs_neither_the_nodes_nor_private_names_of_torch():
    code = ("import sys; sys.path.insert(0, %r)\n"
            "import torch\n"
            "for name in [n for n in vars(torch._C) if n.startswith('_cuda')]: delattr(torch._C, name)\n"
            "import jax_gptq_amd\n"
            "assert 'jax_gptq_amd._torch_experts' not in sys.modules\n") % PACKAGE
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)
