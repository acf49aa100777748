"""What an import of the package needs (no GPU needed)."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

BLOCKED = """
import sys

class NotBuilt:
    def find_spec(self, name, path=None, target=None):
        if name == "bioemu2_b200._training":
            raise ImportError("undefined symbol of another torch")

sys.meta_path.insert(0, NotBuilt())
"""


def run(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)


def test_inference_does_not_need_the_training_extension():
    done = run(BLOCKED + """
import bioemu2_b200 as b
from bioemu2_b200 import *
assert Transition is b.Transition and "training" not in b.__all__ and "Transition" in b.__all__
for use in ("b.training", "from bioemu2_b200 import training", "import bioemu2_b200.training"):
    try:
        exec(use)
    except ImportError as error:
        assert "_training.so" in str(error) and "undefined symbol" in str(error), error
    else:
        raise AssertionError(use)
try:
    b.nothing
except AttributeError:
    print("fine")
""")
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr


def test_training_is_there_with_the_package():
    done = run("from bioemu2_b200 import *\nassert training.Linear and training.LayerNorm\nimport bioemu2_b200 as b\nassert b.training is training")
    assert done.returncode == 0, done.stderr
