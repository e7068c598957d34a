from metellus_amd.compute.serving.serving import ServingFragment

__all__ = ["ServingFragment"]
