"""LeNet for MNIST-shaped inputs (reference: model_ops/lenet.py:12-35)."""

import torch.nn as nn
import torch.nn.functional as F

from ..ops.linear_ops import linear_relu


class LeNet(nn.Module):
    """Two conv + two fc; 28x28 single-channel input by default."""

    linear_relus = ("fc1",)

    def __init__(self, num_classes: int = 10, in_channels: int = 1):
        super().__init__()
        self.conv1 = nn.Conv2d(in_channels, 20, kernel_size=5)
        self.conv2 = nn.Conv2d(20, 50, kernel_size=5)
        self.fc1 = nn.Linear(50 * 4 * 4, 500)
        self.fc2 = nn.Linear(500, num_classes)

    def forward(self, x):
        x = F.max_pool2d(F.relu(self.conv1(x)), 2)
        x = F.max_pool2d(F.relu(self.conv2(x)), 2)
        x = x.flatten(1)
        x = linear_relu(self.fc1, x)
        return self.fc2(x)
