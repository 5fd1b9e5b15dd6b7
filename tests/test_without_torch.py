"""The host-memory calls (forward_host, split_compute, the GGUF readers) need numpy alone: neither
the binding nor the build of the C-ABI library needs torch.  CPU only."""
import os
import subprocess
import sys
import textwrap

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
