"""Refusals of the extension raise, with messages that are whole strings.

The build links libstdc++ into the extension, whose stream formatting of numbers does not work beside the one
that torch loads: a message of several parts of which one is a number ends the process instead of raising."""
import re
from pathlib import Path

import pytest
import torch

CSRC = Path(__file__).resolve().parents[1] / 'deepep_trn_b200' / 'csrc'
needs_cuda = pytest.mark.skipif(not torch.cuda.is_available(), reason='needs CUDA')


def _checks(text):
    """The arguments of every TORCH_CHECK, split at commas outside of brackets and strings."""
    for m in re.finditer(r'TORCH_CHECK\(', text):
        args, depth, quoted, start, i = [], 1, False, m.end(), m.end()
        while depth:
            c = text[i]
            if quoted:
                i += c == '\\'
                quoted = c != '"'
            elif c == '"':
                quoted = True
            elif c in '([{':
                depth += 1
            elif c in ')]}':
                depth -= 1
            elif c == ',' and depth == 1:
                args.append(text[start:i])
                start = i + 1
            i += 1
        yield text[:m.start()].count('\n') + 1, args + [text[start:i - 1]]


def _formats_a_number(part):
    rest = re.sub(r'"(?:\\.|[^"\\])*"', '', part).strip(' \n+')
    return rest != '' and not rest.startswith('std::to_string(') and rest != 'what'   # what: a const char*


def test_scan_finds_what_it_looks_for():
    bad = 'TORCH_CHECK(k < 3, "k, (", k, ")");\nTORCH_CHECK(f(a, b), "plain, " + std::to_string(3), " text");'
    found = [(line, [p for p in args[1:] if _formats_a_number(p)]) for line, args in _checks(bad)]
    assert found == [(1, [' k']), (2, [])]


@pytest.mark.parametrize('path', sorted(p.name for p in CSRC.iterdir() if p.suffix in ('.cu', '.cpp', '.h', '.cuh')))
def test_messages_are_strings(path):
    for line, args in _checks((CSRC / path).read_text()):
        bad = [p for p in args[1:] if _formats_a_number(p)]
        assert not bad, f'{path}:{line}: {bad}'


@pytest.mark.gpu
@needs_cuda
def test_refused_tensor_map_raises():
    from deepep_trn_b200.ops.gemm import grouped_gemm
    A = torch.zeros(1, 64, device='cuda', dtype=torch.bfloat16).as_strided((1, 64), (1 << 40, 1))   # stride past the map's
    B = torch.zeros(1, 64, 64, device='cuda', dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match='failed: 1'):
        grouped_gemm(A, B, torch.tensor([0, 1], device='cuda'))
