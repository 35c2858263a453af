"""The paged cache's operators and the logit rules without a device, at the
edges of what their calls allow: the bounds of lists and rows, and refusals."""
import os
import subprocess


from test_paged import HERE, ROOT


def host_check(tmp_path, name, trials):
    exe = str(tmp_path / name)
    subprocess.run(["g++", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "isa-lm_amd", "csrc"),
                    os.path.join(HERE, "csrc", name + ".cpp"), "-o", exe], check=True)
    r = subprocess.run([exe, str(trials)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("ok"), (r.returncode, r.stdout + r.stderr)


def test_lists_are_read_to_their_counts(tmp_path):
    host_check(tmp_path, "list_bounds", 1000)


def test_negative_rows_are_out_of_range(tmp_path):
    host_check(tmp_path, "row_bounds", 100000)
