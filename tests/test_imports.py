"""What an import of the package needs: neither torch's part of the library nor torch itself where they are not used."""
import subprocess
import sys

import pytest


def run(code):
    return subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)


def test_everything_else_works_without_the_torch_part():
    """_torchcall.so is built for one torch: where it does not fit, only the calls that go through it say so."""
    r = run("import sys; sys.modules['ppo_amd._torchcall'] = None\n"
            "from ppo_amd import *\n"
            "import ppo_amd, torch\n"
            "assert ExperienceBuffer is ppo_amd.ExperienceBuffer and QuantizedRows is ppo_amd.QuantizedRows\n"
            "for call in (lambda: action_stats(torch.zeros(1, 1), torch.zeros(1)), lambda: shape_logits(torch.zeros(1, 1))):\n"
            "    try:\n"
            "        call()\n"
            "    except PpoXpError as e:\n"
            "        assert '_torchcall.so is not built' in str(e), e\n"
            "    else:\n"
            "        raise SystemExit('called')\n")
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("code", ["import ppo_amd", "import ppo_amd; ppo_amd.ExperienceBuffer, ppo_amd.gae_chunk", "from ppo_amd import ExperienceBatcher"])
def test_torch_is_imported_on_first_use(code):
    r = run("import sys; sys.modules['torch'] = None\n" + code)
    assert r.returncode == 0, r.stderr
