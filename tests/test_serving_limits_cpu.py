"""CPU checks of the serving operators at the ends of what they take: records that hold
anything, the largest launches, copies that fail."""
import os
import subprocess


def test_records_of_rows_stay_in_their_slots():
    """What attention over shared prefixes reads back of rows that nothing was left for."""
    cdir = os.path.join(os.path.dirname(__file__), "cpp")
    subprocess.run(["make", "-C", cdir, "attn_row"], check=True, capture_output=True)
    out = subprocess.run([os.path.join(cdir, "attn_row")], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and "wrong 0" in out.stdout, out.stdout
