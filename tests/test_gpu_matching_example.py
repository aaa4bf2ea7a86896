"""The matching operators together with the projectors: examples/classify_images.py on a small set."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_classify_images(gpu):
    spec = importlib.util.spec_from_file_location("classify_images", os.path.join(ROOT, "examples", "classify_images.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.run(box=24, images=300, poses=40, classes=3, noise=1.0)
    # noise of the references' own rms over 600 coefficients: hypotheses lie tens of log units apart
    assert r["class_accuracy"] > 0.95
    assert r["log_prob_of_truth"] > -0.5 and 0 <= r["entropy"] < 0.5
    assert r["map_correlation"] > 0.5
    # the noise is 1 per component; what is left of it lies within the sampling error of 200000 values
    assert 0.9 < r["noise_power"] < 1.2
    assert r["likelihood_gain"] > 0
