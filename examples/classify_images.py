"""Images of several volumes, their classes and poses unknown: scores, posterior, classes, volumes.

The steps between the projection operators, as a user runs them:

  project      every class's volume at every pose of a grid        project_3d_to_2d_forw
  score        every image against every projection, in 8 bits     matching.block_scores
  posterior    log probabilities of the (class, pose) hypotheses   matching.log_probs
  sort         images by the classes of their best hypotheses      matching.sort_by_class, dispatch
  backproject  each class's images, weighted by their posterior    backproject_2d_to_3d_forw, reconstruct
  expect       each class's projections back in image order        project_3d_to_2d_forw, matching.combine
  refine       the volumes by the gradient of the likelihood       matching.log_probs(...).log_sum

Run on a GPU: python examples/classify_images.py [--box 32] [--images 512] [--poses 64] [--classes 3]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "torch-projectors_amd"))
import torch_projectors as tp  # noqa: E402
from torch_projectors import fourier, matching  # noqa: E402

OVERSAMPLING = 2.0


def random_rotations(count, g):
    q = torch.nn.functional.normalize(torch.randn(count, 4, generator=g, device=g.device), dim=1)
    w, x, y, z = q.unbind(1)
    return torch.stack([1 - 2 * (y * y + z * z), 2 * (x * y - z * w), 2 * (x * z + y * w),
                        2 * (x * y + z * w), 1 - 2 * (x * x + z * z), 2 * (y * z - x * w),
                        2 * (x * z - y * w), 2 * (y * z + x * w), 1 - 2 * (x * x + y * y)], 1).view(count, 3, 3)


def random_volume(n, g):
    """A few Gaussian blobs in an n^3 box."""
    at = torch.arange(n, device=g.device) - n / 2
    grid = torch.stack(torch.meshgrid(at, at, at, indexing="ij"), -1)
    centres = (torch.rand(12, 3, generator=g, device=g.device) - 0.5) * n * 0.5
    return sum(torch.exp(-(grid - c).square().sum(-1) / (2 * (n / 16) ** 2)) for c in centres)


def projections(volumes, rotations, n):
    """[C, N, N, N/2+1] at [P, 3, 3] -> [C, P, n, n/2+1]."""
    return tp.project_3d_to_2d_forw(volumes, rotations[None], output_shape=(n, n), oversampling=OVERSAMPLING)


def plane_weights(n, device):
    """Square roots of how often a column of the half plane stands in the whole one."""
    w = torch.full((n // 2 + 1,), 2.0 ** 0.5, device=device)
    w[0] = w[-1] = 1.0
    return w


def run(box=32, images=512, poses=64, classes=3, noise=1.0, seed=0, device="cuda:0"):
    g = torch.Generator(device=device).manual_seed(seed)
    n, w = box, plane_weights(box, device)
    rot = random_rotations(poses, g)
    truth = torch.stack([fourier.to_fourier(random_volume(n, g), OVERSAMPLING) for _ in range(classes)])
    refs = projections(truth, rot, n) * w
    # unit noise where a reference has unit power, times `noise`
    scale = 1.0 / (noise * refs.abs().square().mean().sqrt())
    truth, refs = truth * scale, refs * scale
    is_class = torch.randint(0, classes, (images,), generator=g, device=device)
    is_pose = torch.randint(0, poses, (images,), generator=g, device=device)
    hypothesis = is_class * poses + is_pose
    flat_refs = refs.view(classes * poses, n, n // 2 + 1)
    noise_of = torch.view_as_complex(torch.randn(images, n, n // 2 + 1, 2, generator=g, device=device))
    data = flat_refs[hypothesis] + noise_of
    result = {}

    # score and posterior: log p(image | hypothesis) = <image, ref> - |ref|^2 / 2 + what the image alone decides
    bias = -0.5 * flat_refs.abs().square().sum((1, 2))
    scores = matching.block_scores(data, matching.quantize_blocks(flat_refs), bias=bias)
    post = matching.log_probs(scores, hypothesis, top=2)
    best = post.top_index[:, 0]
    result["class_accuracy"] = (best // poses == is_class).float().mean().item()
    result["log_prob_of_truth"] = post.given.mean().item()
    result["entropy"] = post.entropy.mean().item()

    # each class's images with their weights, in one stretch each
    order = matching.sort_by_class(post.top_index // poses, classes)
    weights = post.top.exp()
    rows = matching.dispatch(data / w, order, weights)
    row_rot = rot[post.top_index % poses].view(-1, 3, 3)[order.order.long()]
    row_weights = weights.view(-1)[order.order.long()][:, None, None].expand(rows.shape).contiguous()
    ends = order.offsets.tolist()
    maps, expected = [], torch.empty_like(rows)
    for c in range(classes):
        part = slice(ends[c], ends[c + 1])
        volume, weight = tp.backproject_2d_to_3d_forw(rows[None, part].contiguous(), row_rot[None, part].contiguous(),
                                                      weights=row_weights[None, part].contiguous(),
                                                      oversampling=OVERSAMPLING)
        maps.append(fourier.reconstruct(volume[0], weight[0], OVERSAMPLING, reg=0.1))
        expected[part] = projections(truth[c:c + 1], row_rot[part], n)[0] if ends[c + 1] > ends[c] else 0
    wanted = torch.stack([fourier.from_fourier(v, OVERSAMPLING) for v in truth])
    got = torch.stack(maps)
    result["map_correlation"] = min(torch.corrcoef(torch.stack([a.flatten(), b.flatten()]))[0, 1].item()
                                    for a, b in zip(got, wanted))

    # the expected projection of every image, and the noise that it leaves
    residual = data - matching.combine(expected, order, weights / weights.sum(1, keepdim=True)) * w
    result["noise_power"] = residual.abs().square().mean().item() / 2

    # one step up the marginal likelihood from blurred volumes
    volumes = (0.8 * truth).requires_grad_()
    real_data = torch.view_as_real(data).reshape(images, -1)

    def likelihood(v):
        r = torch.view_as_real(projections(v, rot, n) * w).reshape(classes * poses, -1)
        return matching.log_probs(real_data @ r.t() - 0.5 * r.square().sum(1)).log_sum.mean()

    before = likelihood(volumes)
    (slope,) = torch.autograd.grad(before, volumes)
    step = 0.1 * volumes.detach().norm() / slope.norm()
    with torch.no_grad():
        result["likelihood_gain"] = (likelihood(volumes + step * slope) - before).item()
    return result


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--box", type=int, default=32)
    ap.add_argument("--images", type=int, default=512)
    ap.add_argument("--poses", type=int, default=64)
    ap.add_argument("--classes", type=int, default=3)
    ap.add_argument("--noise", type=float, default=1.0, help="noise amplitude per Fourier coefficient, in reference rms")
    a = ap.parse_args()
    for name, value in run(a.box, a.images, a.poses, a.classes, a.noise).items():
        print(f"{name:20s} {value:.4f}")


if __name__ == "__main__":
    main()
