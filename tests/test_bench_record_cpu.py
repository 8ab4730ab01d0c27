"""A committed measurement of the GEMM kernel is taken for what bench.py runs only if it was taken on the same sources and flags."""
import shutil

import bench
from mmmm_amd import build


def test_the_digest_follows_sources_and_flags_not_the_version_number(tmp_path, monkeypatch):
    (tmp_path / 'mmmm_amd').mkdir()
    shutil.copytree(bench.ROOT / 'mmmm_amd' / 'csrc', tmp_path / 'mmmm_amd' / 'csrc')
    here = bench.gemm_source_digest()
    monkeypatch.setattr(bench, 'ROOT', tmp_path)
    assert bench.gemm_source_digest() == here
    gemm = tmp_path / 'mmmm_amd' / 'csrc' / 'gemm.hip'
    text = gemm.read_text()
    assert text.count('\nint vm_version(void)') == 1
    gemm.write_text(text.replace('int vm_version(void) { return', 'int vm_version(void) { return 1 +'))
    assert bench.gemm_source_digest() == here
    gemm.write_text(text + '\n')
    assert bench.gemm_source_digest() != here
    gemm.write_text(text)
    monkeypatch.setattr(build, 'CFLAGS', build.CFLAGS[:-1])
    assert bench.gemm_source_digest() != here
