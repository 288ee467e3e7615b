"""Where the reference's sources are looked for: a directory that does not hold them
counts as no tree, so that the build and the oracle tests go on without it."""
from oracle import c_oracle


def test_a_directory_without_the_sources_is_no_tree(tmp_path, monkeypatch):
    monkeypatch.setenv("FA_REFERENCE_TREE", str(tmp_path))
    assert c_oracle.reference_tree() is None
    (tmp_path / "attention.cu").write_text("")
    assert c_oracle.reference_tree() is None
    (tmp_path / "bwd.cu").write_text("")
    assert c_oracle.reference_tree() == str(tmp_path)
    monkeypatch.setenv("FA_REFERENCE_TREE", str(tmp_path / "missing"))
    assert c_oracle.reference_tree() is None
