"""Small programs that use the package as a serving program would: `python -m orbitquant_amd.examples.decode`."""
