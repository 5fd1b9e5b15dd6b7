"""The host-memory calls (forward_host, split_compute, the GGUF readers) need numpy alone: neither
the binding nor the build of the C-ABI library needs torch.  CPU only."""
import os
import shutil
import subprocess
import sys
import textwrap

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(REPO, "llama-sandbox_amd")

# moe_block with a library that only hands out a context: what the constructor itself does
STUB = textwrap.dedent("""
    import sys
    sys.path.insert(0, sys.argv[1])
    import moe_block as mb

    class Lib:
        made = freed = 0
        def moe_ctx_create(self, device, budget, out):
            Lib.made += 1
            out._obj.value = 4096
            return 0
        def moe_ctx_destroy(self, h):
            Lib.freed += 1

    mb.load_library = lambda path=None: Lib()
""")


def run(code):
    r = subprocess.run([sys.executable, "-c", STUB + textwrap.dedent(code), PKG], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout.split()


def test_a_context_is_made_where_torch_is_absent():
    out = run("""
        sys.modules["torch"] = None  # any import of it raises ModuleNotFoundError
        with mb.MoeBlock(0) as b:
            print(b.h, b.device)
        print(Lib.made, Lib.freed)
    """)
    assert out == ["4096", "0", "1", "1"]


def test_a_context_does_not_import_torch():
    """It takes seconds and hundreds of MB, and a caller with host arrays has no use for it."""
    out = run("""
        b = mb.MoeBlock(0)
        print("torch" in sys.modules)
        b.close()
    """)
    assert out == ["False"]


def test_the_operators_say_that_they_take_torch_tensors():
    out = run("""
        import numpy as np
        sys.modules["torch"] = None
        b, x = mb.MoeBlock(0), np.zeros((2, 8), np.float32)
        calls = [lambda: b.dispatch(x, x, x), lambda: b.dispatch_grad(x, x, x), lambda: b.combine(x, x, x, x),
                 lambda: b.combine_grad(x, x, x, x, x, x), lambda: b.quantize_i8(x, x, x),
                 lambda: b.matmul_i8(x, x, x, x, x)]
        for call in calls:
            try:
                call()
            except ValueError as e:
                print("torch" in str(e))
    """)
    assert out == ["True"] * 6


@pytest.fixture
def tree(tmp_path):
    """A copy of what make reads, with stand-ins for the compilers that write their output, and a python3
    whose torch is missing."""
    pkg = tmp_path / "pkg"
    shutil.copytree(PKG, pkg, ignore=shutil.ignore_patterns("*.so", "*.o", "moe-server", "__pycache__"))
    shutil.copytree(os.path.join(REPO, "include"), tmp_path / "include")
    tools = tmp_path / "tools"
    tools.mkdir()
    # a compiler that cannot find torch's headers unless it is told where they are
    compiler = """#!/bin/sh
case "$*" in *moe_torch.cpp*) case "$*" in *-I/torch/include*) ;; *) echo "no torch headers" >&2; exit 1 ;; esac ;; esac
while [ $# -gt 0 ]; do [ "$1" = -o ] && echo built > "$2"; shift; done
"""
    for name, text in (("hipcc", compiler), ("g++", compiler),
                       ("python3", "#!/bin/sh\necho \"No module named 'torch'\" >&2\nexit 1\n")):
        (tools / name).write_text(text)
        (tools / name).chmod(0o755)

    def make(*args):
        env = dict(os.environ, PATH=f"{tools}:{os.environ['PATH']}", HIPCC=str(tools / "hipcc"))
        for v in ("MAKEFLAGS", "MAKELEVEL", "MFLAGS"):
            env.pop(v, None)
        return subprocess.run(["make", "-C", str(pkg), *args], env=env, capture_output=True, text=True)

    make.pkg, make.tools = pkg, tools
    return make


@pytest.mark.parametrize("args", [(), ("-j8",), ("-s", "-B")])
def test_make_builds_the_library_without_torch(tree, args):
    r = tree(*args)
    assert r.returncode == 0, r.stderr
    assert (tree.pkg / "libmoe_block.so").exists() and (tree.pkg / "moe-server").exists()
    assert not (tree.pkg / "moe_torch.so").exists()


def test_a_module_that_no_longer_builds_is_not_left_behind(tree):
    (tree.pkg / "moe_torch.so").write_text("of another source")
    assert tree("-B").returncode == 0
    assert not (tree.pkg / "moe_torch.so").exists()


def test_make_builds_the_module_where_torch_is_found_and_its_target_fails_where_not(tree):
    assert tree("moe_torch.so").returncode != 0
    (tree.tools / "python3").write_text("#!/bin/sh\necho -I/torch/include\n")
    r = tree()
    assert r.returncode == 0, r.stderr
    assert (tree.pkg / "moe_torch.so").exists()
