"""The build's rules from a clean checkout: every product that `make` links makes the directory it goes to, whichever
other rules have run by then."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "fercuda_b200" / "csrc"
PRODUCTS = ["libptx_core.so", "libptx_kernels.so", "libfercuda_capi.so", "libfercuda_bench.so", "libptx_hook.so",
            "fer_alloc_bench"]


def _make(out, *args):
    return subprocess.run(["make", "-C", str(CSRC), f"OUT={out}", f"OBJ={out.parent}/obj", *args], capture_output=True, text=True)


def test_the_list_of_products(tmp_path):
    out = tmp_path / "lib"
    run = _make(out, "-n", "all")
    assert run.returncode == 0, run.stderr
    linked = {p.name for p in map(Path, run.stdout.split()) if p.parent == out}
    assert set(PRODUCTS) <= linked and linked <= set(PRODUCTS)


@pytest.mark.parametrize("product", PRODUCTS)
def test_a_product_makes_its_directory(tmp_path, product):
    """Of a product and what it is made from alone: the directory comes before the first that is written there."""
    out = tmp_path / "lib"
    run = _make(out, "-n", f"{out}/{product}")
    assert run.returncode == 0, run.stderr
    text = run.stdout
    made, written = text.find(f"mkdir -p {out}\n"), text.find(f"-o {out}/")
    assert 0 <= made < written


def test_the_allocator_benchmark_builds_alone(tmp_path):
    out = tmp_path / "lib"
    run = _make(out, f"{out}/fer_alloc_bench")
    assert run.returncode == 0, run.stdout + run.stderr
    assert (out / "fer_alloc_bench").is_file()
